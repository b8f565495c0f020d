// Attention of single new tokens over pages of a KV cache: what paged_attention.cu computes, for calls without masks and with at most 16 query heads per kv head that say of their requests that
// each has at most one (max_new 1), or say nothing and have no more tokens than requests.  Right for any number of them, whatever was said.
//
// A tile is one token's heads of one kv head's group, at most 16 rows.  It is bound by HBM, and where a call is small by the time from its launch to its last store; the fifth-generation tensor
// core, whose tiles have 128 rows and whose set-up (tensor memory, barriers, maps) takes microseconds, has nothing to give here.  So, as for the contiguous cache (attention.cu):
//
//   * a warp takes every fourth run of 16 keys and fetches it by cp.async into a ring of its own, so that no warp waits for another before the end of a tile; 96 KiB of ring a CTA, two CTAs
//     an SM.  The pages' numbers come from the table 32 at a time, a lane for each, one batch ahead.
//   * scores and outputs are mma.sync.m16n8k16 with the heads as rows: the score fragment of a warp is, register for register, the operand of the second product.
//   * every row sees all of its keys, so nothing is masked but the last run's end, whose rows are filled with zeros and not read.
//   * equal shares of the line of all tiles, and the join of parts, are those of paged_attention.cu.
//
// fp32 scores, running maxima and sums; probabilities are rounded to the operands' type for the second product, in fp16 times 2^8.
//
// Measured, 64 / 8 heads of 128, pages of 64: 32 requests of 30 to 4000 keys 39.6 us (194 MB: 4.9 TB/s), of 2049 48.3 (5.6 TB/s), of 300 10.4; 4 of 129 keys, 16 / 4 heads, 5.3.  The tensor-core kernel takes 42.7
// and 9.7 for the first and 4 x 100 to 300.  Behind HBM stand 5 us for the shares of the CTAs, the cold ring of each of their tiles, and the join.
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/gpuk_b200.h"
#include "common.cuh"
#include "launch.cuh"
#include "paged_share.cuh"

namespace gpuk {
namespace {

constexpr int kWarps = kDecodeThreads / 32;
constexpr int kRun = 16;                         // keys a warp takes at a time

template <int HD>
constexpr int kStages = 384 / HD;                // runs in a warp's ring: 24 KiB of it, keys and values
template <int HD>
constexpr int kRingBytes = kWarps * kStages<HD> * 2 * kRun * HD * 2;
template <int HD>
constexpr int kPitch = HD + 4;                   // floats of a row of a warp's outputs
static_assert(kWarps * kDecodeGroup * kPitch<128> * 4 <= kRingBytes<128> && kWarps * kDecodeGroup * kPitch<64> * 4 <= kRingBytes<64>, "the warps' outputs reuse the ring");

struct Stats {
    float m[kWarps][kDecodeGroup], l[kWarps][kDecodeGroup];
};

__device__ __forceinline__ void cp_async16(uint32_t to, const void *from, bool there, uint64_t policy) {
    const int bytes = there ? 16 : 0;
    asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(to), "l"(from), "r"(bytes), "l"(policy) : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16 *) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half *) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Where no tile is cut, a CTA takes one, and finds it without the line of all tiles: token blockIdx.x / kv_heads, most often that of the request of the same number.  One warp.
__device__ void find_token(const PagedAttentionParams &p, Start *out) {
    const int lane = threadIdx.x & 31, token = blockIdx.x / p.kv_heads;
    Request r = {};
    if (token < p.batch) r = request_of(p, token);
    int request = token;
    if (token >= p.batch || r.start != token || r.n != 1) {      // the request is the number of those that end in front of the token
        int ended = 0;
        for (int i = lane; i < p.batch; i += 32) ended += p.starts[i + 1] <= token;
        request = __reduce_add_sync(0xffffffffu, ended);
        r.n = 0;
        if (request < p.batch) r = request_of(p, request);
    }
    if (lane == 0) {
        const int tile = token - r.start;
        const bool there = tile >= 0 && tile < r.n;
        out->r = r, out->request = request, out->kvh = blockIdx.x % p.kv_heads, out->tile = tile, out->pos = 0, out->ctas = gridDim.x;
        out->x[0] = 0, out->x[1] = there ? weight_of(p, r, tile) : 0;
    }
}

template <typename T, int HD>
__global__ void __launch_bounds__(kDecodeThreads, kCtasPerSm) paged_decode_kernel(const __grid_constant__ PagedAttentionParams p) {
    constexpr int kChunks = HD / 8, kRowsAtOnce = 32 / kChunks, kCopies = kRun / kRowsAtOnce;      // 16-byte chunks of a row, rows and copies of a warp's pass over a run
    constexpr int kRowBytes = HD * 2, kTileBytes = kRun * kRowBytes, STAGES = kStages<HD>;
    extern __shared__ __align__(128) unsigned char dyn[];
    __shared__ Start start;
    __shared__ Stats st;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    grid_dependency_sync();
    if (!p.may_split) {
        if (warp == 0) find_token(p, &start);
    } else if (warp < 2) {
        find_border(p, &start, warp);
    }
    __syncthreads();
    Joint joint;
    joint.open.slot = -1, joint.head = start.x[1] > start.x[0] ? 3 : 0, joint.ctas = start.ctas;
    const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(dyn)) + warp * (STAGES * 2 * kTileBytes);
    const uint64_t once = policy_once();
    // 16-byte chunk c of row r lies at c ^ (r & 7): the eight rows of an ldmatrix are in different banks
    auto swizzled = [](int r, int c) { return r * kRowBytes + ((c ^ (r & 7)) << 4); };
    const int64_t lane_at = lane / kChunks * p.row_stride + lane % kChunks * 8;      // of the lane's first copy in a run, and where its row goes
    const uint32_t lane_to = lane / kChunks * kRowBytes;
    const int page_mask = (1 << p.page_shift) - 1, per_run = p.page_shift < 4 ? kRun >> p.page_shift : 1;      // pages of a run

    Walk walk(start);
    Segment u;
    bool begins, ends;
    while (walk.next(p, &u, &begins, &ends)) {
        if (!begins) joint.head = ends ? 2 : 1;
        if (begins && !ends) joint.open = u;
        const int token = u.start + u.tok0;
        const int hi = static_cast<int>(min(keys_of(p, walk.r, u.tok0), (static_cast<int64_t>(u.first) + u.blocks) * kKeys)), lo = u.first * kKeys;
        const int runs = (hi - lo + kRun - 1) / kRun, mine = warp < runs ? (runs - warp + kWarps - 1) / kWarps : 0;      // this warp's: warp, warp + 4, ...
        const int32_t *table = p.tables + u.request * p.table_stride;
        const T *kbase = static_cast<const T *>(p.k) + u.kvh * p.head_stride, *vbase = static_cast<const T *>(p.v) + u.kvh * p.head_stride;
        // lane l of a batch: page l % per_run of run l / per_run
        const int batch_runs = 32 / per_run;
        auto pages_from = [&](int i) {
            const int run = i + lane / per_run;
            const int key = lo + (warp + run * kWarps) * kRun + (lane % per_run << p.page_shift);
            return run < mine && key < hi ? table[key >> p.page_shift] : -1;
        };
        int pages = pages_from(0), pages_next = pages_from(batch_runs), issued = 0, in_batch = 0;
        auto issue = [&]() {
            if (issued < mine) {
                if (in_batch == batch_runs) pages = pages_next, pages_next = pages_from(issued + batch_runs), in_batch = 0;
                const uint32_t slot = ring + (issued % STAGES) * (2 * kTileBytes);
                const int row0 = lo + (warp + issued * kWarps) * kRun;
                if (per_run == 1) {      // the run is in one page: an addition for each copy
                    const int page = __shfl_sync(0xffffffffu, pages, in_batch);
                    const bool there = page >= 0 && page < p.num_pages;
                    const int64_t first = there ? page * p.page_stride + (row0 & page_mask) * p.row_stride : 0;
                    const T *k = kbase + first + lane_at, *v = vbase + first + lane_at;
                    const int rows = there ? hi - row0 - lane / kChunks : 0;      // of the lane's, those that are keys
#pragma unroll
                    for (int j = 0; j < kCopies; ++j) {
                        const int r = j * kRowsAtOnce;
                        const uint32_t to = slot + r * kRowBytes + lane_to + (((lane % kChunks) ^ ((r + lane / kChunks) & 7)) << 4);
                        const bool key = r < rows;
                        cp_async16(to, key ? k + r * p.row_stride : kbase, key, once);
                        cp_async16(to + kTileBytes, key ? v + r * p.row_stride : vbase, key, once);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < kCopies; ++j) {
                        const int r = j * kRowsAtOnce + lane / kChunks, c = lane % kChunks, key = row0 + r;
                        const int page = __shfl_sync(0xffffffffu, pages, in_batch * per_run + (r >> p.page_shift));
                        const bool there = key < hi && page >= 0 && page < p.num_pages;
                        const int64_t off = there ? page * p.page_stride + (key & page_mask) * p.row_stride + c * 8 : 0;
                        cp_async16(slot + swizzled(r, c), kbase + off, there, once);
                        cp_async16(slot + kTileBytes + swizzled(r, c), vbase + off, there, once);
                    }
                }
                ++in_batch;
            }
            ++issued;
            asm volatile("cp.async.commit_group;" ::: "memory");      // an empty group past the end keeps the count uniform
        };
#pragma unroll
        for (int i = 0; i < STAGES - 1; ++i) issue();

        // the group's query heads as the rows of the first operand, zero rows beyond them
        uint32_t qa[HD / 16][4];
        const T *qbase = static_cast<const T *>(p.q) + static_cast<int64_t>(token) * p.q_token + static_cast<int64_t>(u.kvh) * p.group * p.q_head;
#pragma unroll
        for (int s = 0; s < HD / 16; ++s)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = g + (r & 1) * 8, col = s * 16 + 2 * t + (r >> 1) * 8;
                qa[s][r] = row < p.group ? *reinterpret_cast<const uint32_t *>(qbase + row * p.q_head + col) : 0u;
            }
        float o[HD / 8][4];
#pragma unroll
        for (int j = 0; j < HD / 8; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[j][e] = 0.f;
        // rows g and g + 8: a warp without a run has seen nothing
        float m[2] = {mine ? kSeen : kLowest, mine ? kSeen : kLowest}, l[2] = {0.f, 0.f};

        for (int i = 0; i < mine; ++i) {
            issue();
            asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
            __syncwarp();
            const uint32_t ks = ring + (i % STAGES) * (2 * kTileBytes), vs = ks + kTileBytes;
            float sc[2][4] = {};
            const int mi = lane >> 3, mr = lane & 7;      // which of the four 8x8 matrices this lane addresses, and its row
#pragma unroll
            for (int s = 0; s < HD / 16; ++s) {
                uint32_t kb[4];      // keys 0-7 | 8-15, dimensions 0-7 | 8-15 of this step
                ldmatrix4(kb, ks + swizzled((mi >> 1) * 8 + mr, 2 * s + (mi & 1)));
                mma(sc[0], qa[s], kb[0], kb[1], static_cast<T *>(nullptr));
                mma(sc[1], qa[s], kb[2], kb[3], static_cast<T *>(nullptr));
            }
            const int row0 = lo + (warp + i * kWarps) * kRun;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[h][e] = row0 + h * 8 + 2 * t + (e & 1) < hi ? sc[h][e] * p.scale_log2 : -INFINITY;
            float mx[2], fade[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                mx[r] = fmaxf(fmaxf(sc[0][2 * r], sc[0][2 * r + 1]), fmaxf(sc[1][2 * r], sc[1][2 * r + 1]));
                mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
                mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
                mx[r] = fmaxf(mx[r], m[r]);
                fade[r] = exp2f(m[r] - mx[r]);
            }
            if (__any_sync(0xffffffffu, mx[0] != m[0] || mx[1] != m[1])) {
#pragma unroll
                for (int j = 0; j < HD / 8; ++j) {
                    o[j][0] *= fade[0], o[j][1] *= fade[0];
                    o[j][2] *= fade[1], o[j][3] *= fade[1];
                }
                l[0] *= fade[0], l[1] *= fade[1];
                m[0] = mx[0], m[1] = mx[1];
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[h][e] = exp2f(sc[h][e] - m[e >> 1] + Half<T>::kBias);
            l[0] += (sc[0][0] + sc[0][1]) + (sc[1][0] + sc[1][1]);
            l[1] += (sc[0][2] + sc[0][3]) + (sc[1][2] + sc[1][3]);
            const uint32_t pa[4] = {Half<T>::pack(sc[0][0], sc[0][1]), Half<T>::pack(sc[0][2], sc[0][3]), Half<T>::pack(sc[1][0], sc[1][1]), Half<T>::pack(sc[1][2], sc[1][3])};
#pragma unroll
            for (int j = 0; j < HD / 16; ++j) {
                uint32_t vb[4];      // keys 0-7 | 8-15 of dimensions 0-7, then of dimensions 8-15
                ldmatrix4_trans(vb, vs + swizzled((mi & 1) * 8 + mr, 2 * j + (mi >> 1)));
                mma(o[2 * j], pa, vb[0], vb[1], static_cast<T *>(nullptr));
                mma(o[2 * j + 1], pa, vb[2], vb[3], static_cast<T *>(nullptr));
            }
            __syncwarp();      // the next issue refills the slot of the run before this one: every lane is past it
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
            if (t == 0) st.m[warp][g + 8 * r] = m[r], st.l[warp][g + 8 * r] = l[r];
        }
        __syncthreads();      // all warps are done with the ring: it takes their outputs, a tile of [16][pitch] each
        float *tiles = reinterpret_cast<float *>(dyn);
#pragma unroll
        for (int j = 0; j < HD / 8; ++j)
#pragma unroll
            for (int r = 0; r < 2; ++r)
                if (g + 8 * r < p.group)
                    *reinterpret_cast<float2 *>(tiles + (warp * kDecodeGroup + g + 8 * r) * kPitch<HD> + j * 8 + 2 * t) = make_float2(o[j][2 * r], o[j][2 * r + 1]);
        __syncthreads();
        // four outputs a thread: the warps' in units of the largest maximum, in their order
        for (int e = tid; e < p.group * (HD / 4); e += kDecodeThreads) {
            const int h = e / (HD / 4), d = e % (HD / 4) * 4;
            float top = st.m[0][h], total = 0.f;
#pragma unroll
            for (int w = 1; w < kWarps; ++w) top = fmaxf(top, st.m[w][h]);
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float4 v = *reinterpret_cast<const float4 *>(tiles + (w * kDecodeGroup + h) * kPitch<HD> + d);
                const float f = exp2f(st.m[w][h] - top);
                acc.x += f * v.x, acc.y += f * v.y, acc.z += f * v.z, acc.w += f * v.w;
                total += f * st.l[w][h];
            }
            if (u.slot < 0) {
                // all scores -infinity: NaN, as a softmax has it
                const float r = total == 0.f ? __int_as_float(0x7fffffff) : 1.f / total;
                *reinterpret_cast<uint2 *>(static_cast<T *>(p.out) + static_cast<int64_t>(token) * p.out_token + (static_cast<int64_t>(u.kvh) * p.group + h) * p.out_head + d) =
                    make_uint2(Half<T>::pack(acc.x * r, acc.y * r), Half<T>::pack(acc.z * r, acc.w * r));
            } else {
                reinterpret_cast<float4 *>(p.partial)[(static_cast<int64_t>(u.slot) * (HD / 4) + d / 4) * kRows + h] = acc;
                if (d == 0) {
                    float *stats = p.stats + static_cast<int64_t>(u.slot) * 2 * kRows + h;
                    stats[0] = top, stats[kRows] = total;
                }
            }
        }
        __syncthreads();      // the next tile's copies go where these outputs were
    }
    if (tid == 0 && p.may_split) p.joints[blockIdx.x] = joint;
}

template <typename T, int HD>
const void *kernel_of(int *smem) {
    *smem = kRingBytes<HD>;
    return reinterpret_cast<const void *>(&paged_decode_kernel<T, HD>);
}

}  // namespace

const void *paged_decode_of(int dtype, int head_dim, int *smem) {
    if (dtype == GPUK_DTYPE_BF16) return head_dim == 128 ? kernel_of<__nv_bfloat16, 128>(smem) : kernel_of<__nv_bfloat16, 64>(smem);
    return head_dim == 128 ? kernel_of<__half, 128>(smem) : kernel_of<__half, 64>(smem);
}

}  // namespace gpuk
