// What keeps a paged KV cache between the passes of attention over it, one launch each:
//
//   plan_kernel   block tables made to fit the requests' lengths, and for each new token its position, its slot and, in a tree of drafts, its ancestors.
//   keep_kernel   the keys and values of a tree's accepted path moved to the end of the cached tokens, in all layers.
//
// Both move little and are bound by latency: a plan is one cluster that reads the lengths once and meets once, in place of the dozens of operators (prefix sums, searches,
// scatters) that it takes otherwise; the moves of a path read eight rows ahead of their writes.  Measured: 256 trees of 17 to 64 nodes 8.4 us, 48 prompts of 72 000 tokens 11.7; paths of 64 trees in
// four layers and of 4 trees in two 4.3 us call after call, which is the host's time, and 3.1 and 2.1 from a graph.  A plan's walk from a node to its root is in shared memory and a mask of 64 bits: in global memory and eight words it took the same trees 12.9 us.
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/gpuk_b200.h"
#include "common.cuh"
#include "launch.cuh"
#include "linear.cuh"

namespace gpuk {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWarps = kPlanThreads / 32;
constexpr int kMaxRequests = 4096;
constexpr int kMaxWords = 8;

struct PlanParams {
    const int32_t *lens, *new_lens, *held, *free_count, *parents;
    int32_t *tables, *free;
    int32_t *starts, *masks, *held_out, *free_count_out;
    int64_t *positions, *slots;
    int64_t table_stride;
    int batch, width, page_shift, capacity, total, words;
};

// Sums over the threads in front, and over all of them, that stay at a ceiling once they reach it.
constexpr int kCeiling = 0x3fffffff;
struct Saturated {
    int v;
    __device__ Saturated operator+(Saturated o) const { return {min(v + o.v, kCeiling)}; }
    __device__ Saturated up(int lanes) const { return {__shfl_up_sync(0xffffffffu, v, lanes)}; }
    __device__ Saturated at(int lane) const { return {__shfl_sync(0xffffffffu, v, lane)}; }
};
// Two sums at once, each below 2^31.
struct Pair {
    int a, b;
    __device__ Pair operator+(Pair o) const { return {a + o.a, b + o.b}; }
    __device__ Pair up(int lanes) const { return {__shfl_up_sync(0xffffffffu, a, lanes), __shfl_up_sync(0xffffffffu, b, lanes)}; }
    __device__ Pair at(int lane) const { return {__shfl_sync(0xffffffffu, a, lane), __shfl_sync(0xffffffffu, b, lane)}; }
};
template <typename V>
__device__ V warp_upto(V v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const V t = v.up(o);
        if (lane >= o) v = v + t;
    }
    return v;
}
// `before`: the sum of the threads in front; returns that of all.
template <typename V>
__device__ V block_before(V v, V *before, V (&warp_sums)[kPlanWarps + 1]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const V upto = warp_upto(v), front = upto.up(1);
    __syncthreads();      // the sums have been read
    if (lane == 31) warp_sums[warp] = upto;
    __syncthreads();
    const V sums = warp_upto(warp_sums[lane]), others = sums.at(max(warp - 1, 0)), all = sums.at(31);
    *before = warp == 0 ? V{} : others;
    if (lane > 0) *before = *before + front;
    return all;
}

// Parents that a CTA keeps at hand beside those of its tokens: of the request that goes on from in front of them.
constexpr int kBehind = 256;
constexpr int kPlanCtas = 16;      // of a cluster, where it has a place

// The mask of a token: `WORDS` words of 32 bits, two of them as one of 64, none without parents.
template <int WORDS>
struct Mask {
    uint32_t w[WORDS] = {};
    __device__ void add(int node) {
#pragma unroll
        for (int i = 0; i < WORDS; ++i)
            if (i == node >> 5) w[i] |= 1u << (node & 31);
    }
    __device__ uint32_t word(int i) const { return w[i]; }
};
template <>
struct Mask<0> {
    __device__ void add(int) {}
    __device__ uint32_t word(int) const { return 0; }
};
template <>
struct Mask<2> {
    uint64_t w = 0;
    __device__ void add(int node) { w |= node < 64 ? 1ull << node : 0ull; }
    __device__ uint32_t word(int i) const { return static_cast<uint32_t>(w >> 32 * i); }
};

template <int WORDS>
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const __grid_constant__ PlanParams p) {
    constexpr int kTokens = WORDS ? 2 : 4, kSpan = kTokens * kPlanThreads;      // that a thread places at a time, and a CTA
    extern __shared__ int32_t lists[];      // per request: first token, cached tokens, the pages in front that come back or go out, and those that it holds
    __shared__ Saturated token_sums[kPlanWarps + 1];
    __shared__ Pair page_sums[kPlanWarps + 1];
    __shared__ int32_t family[WORDS ? kSpan + kBehind : 1];
    __shared__ unsigned long long over;      // pages for which the rows of the table have no room
    int32_t *const starts = lists, *const lens = starts + p.batch + 1, *const back_at = lens + p.batch, *const want_at = back_at + p.batch, *const holds = want_at + p.batch;
    const int ctas = cluster_size(), cta = cluster_cta_rank(), tid = threadIdx.x, lane = tid & 31;
    const int thread = cta * kPlanThreads + tid, threads = ctas * kPlanThreads;
    if (tid == 0) over = 0;
    grid_dependency_sync();
    const int64_t room = static_cast<int64_t>(p.width) << p.page_shift;
    const int page = 1 << p.page_shift;
    auto stage_family = [&](int base) {
        if (WORDS == 0) return;
#pragma unroll
        for (int i = 0; i < (kSpan + kBehind + kPlanThreads - 1) / kPlanThreads; ++i) {
            const int at = i * kPlanThreads + tid, t = base - kBehind + at;
            if (at < kSpan + kBehind) family[at] = t >= 0 && t < p.total ? p.parents[t] : -1;
        }
    };
    stage_family(cta * kSpan);

    struct Need {
        int held, need;
    };
    auto pages_of = [&](int i, int n) { return (static_cast<int64_t>(lens[i]) + n + page - 1) >> p.page_shift; };
    auto need_of = [&](int i) { return Need{holds[i], static_cast<int>(min(pages_of(i, starts[i + 1] - starts[i]), static_cast<int64_t>(p.width)))}; };
    // every CTA goes over all requests: starts, and how many pages come back and go out in front of each
    Saturated tokens = {};
    Pair pages = {};
    for (int base = 0; base < p.batch; base += kPlanThreads) {
        const int i = base + tid;
        const bool here = i < p.batch;
        const int n_given = here ? min(max(p.new_lens[i], 0), kCeiling) : 0, cached = here ? max(p.lens[i], 0) : 0, held = here ? min(max(p.held[i], 0), p.width) : 0;
        Saturated front;
        const Saturated all = block_before(Saturated{n_given}, &front, token_sums);
        const int first = min((tokens + front).v, p.total), n = min(n_given, p.total - first);
        tokens = tokens + all;
        Pair v = {};
        if (here) {
            starts[i] = first, lens[i] = cached, holds[i] = held;
            const int64_t want = pages_of(i, n);
            const int need = static_cast<int>(min(want, static_cast<int64_t>(p.width)));
            v = {max(held - need, 0), max(need - held, 0)};
            if (want > need) atomicAdd(&over, static_cast<unsigned long long>(want - need));
        }
        Pair before;
        const Pair sum = block_before(v, &before, page_sums);
        if (here) back_at[i] = pages.a + before.a, want_at[i] = pages.b + before.b;
        pages = pages + sum;
    }
    if (tid == 0) starts[p.batch] = min(tokens.v, p.total);
    const int count = min(max(p.free_count[0], 0), p.capacity);
    const int there = static_cast<int>(min(static_cast<int64_t>(count) + pages.a, static_cast<int64_t>(p.capacity)));
    __syncthreads();
    // pages that are too many, onto the list: a warp per request
    for (int i = thread / 32; i < p.batch; i += threads / 32) {
        const Need r = need_of(i);
        for (int j = r.need + lane; j < r.held; j += 32) {
            const int64_t at = static_cast<int64_t>(count) + back_at[i] + j - r.need;
            if (at < p.capacity) p.free[at] = p.tables[i * p.table_stride + j];
        }
    }
    cluster_arrive();
    auto page_from = [&](int i, int nth) {
        const int64_t at = static_cast<int64_t>(there) - 1 - (static_cast<int64_t>(want_at[i]) + nth);
        return at >= 0 ? p.free[at] : -1;
    };
    // positions, slots and ancestors: a CTA takes every so many spans of tokens
    const int seen = starts[p.batch];
    int top = 1;
    while (top * 2 < p.batch) top *= 2;
    bool met = false;
    for (int64_t span = static_cast<int64_t>(cta) * kSpan; span < p.total; span += static_cast<int64_t>(ctas) * kSpan) {
        const int base = static_cast<int>(span);
        if (met) {
            __syncthreads();      // those of the last span have been read
            stage_family(base);
            __syncthreads();
        }
        int request[kTokens] = {};      // the last whose first token is not behind
        for (int step = top; step > 0; step >>= 1)
#pragma unroll
            for (int k = 0; k < kTokens; ++k)
                if (request[k] + step < p.batch && starts[request[k] + step] <= base + k * kPlanThreads + tid) request[k] += step;
        if (!met) cluster_wait();      // the list is whole, and everybody has read the counts: they may be written where they came from
        met = true;
        int32_t id[kTokens];
#pragma unroll
        for (int k = 0; k < kTokens; ++k) {
            const int t = base + k * kPlanThreads + tid;
            id[k] = -1;
            if (t >= seen) continue;
            const int64_t at = static_cast<int64_t>(lens[request[k]]) + t - starts[request[k]];
            if (at >= room) continue;
            const int block = static_cast<int>(at >> p.page_shift), held = holds[request[k]];
            id[k] = block < held ? p.tables[request[k] * p.table_stride + block] : page_from(request[k], block - held);
        }
#pragma unroll
        for (int k = 0; k < kTokens; ++k) {
            const int t = base + k * kPlanThreads + tid;
            if (t >= p.total) continue;
            int64_t position = -1, slot = -1;
            Mask<WORDS> mask;
            if (t < seen) {
                const int first = starts[request[k]], index = t - first;
                position = static_cast<int64_t>(lens[request[k]]) + index;
                if (id[k] >= 0) slot = (static_cast<int64_t>(id[k]) << p.page_shift) + (position & (page - 1));
                if (WORDS) {
                    // each parent comes before its child, so the walk ends; any other number is no parent
                    const int at = first - base + kBehind;
                    int depth = 0;
                    for (int node = index;;) {
                        mask.add(node);
                        const int up = at + node >= 0 ? family[at + node] : p.parents[first + node];
                        if (up < 0 || up >= node) break;
                        node = up;
                        ++depth;
                    }
                    position = static_cast<int64_t>(lens[request[k]]) + depth;
                }
            }
            p.positions[t] = position;
            p.slots[t] = slot;
            if (WORDS)
#pragma unroll
                for (int w = 0; w < WORDS; ++w)
                    if (w < p.words) p.masks[static_cast<int64_t>(t) * p.words + w] = static_cast<int32_t>(mask.word(w));
        }
    }
    if (!met) cluster_wait();
    // the tables' new ends and what the requests hold
    for (int i = thread / 32; i < p.batch; i += threads / 32) {
        const Need r = need_of(i);
        const int want = max(r.need - r.held, 0);
        for (int j = lane; j < want; j += 32) p.tables[i * p.table_stride + r.held + j] = page_from(i, j);
        if (lane == 0) {
            p.held_out[i] = min(r.held, r.need) + min(want, max(there - want_at[i], 0));
            p.starts[i] = starts[i];
        }
    }
    if (thread == 0) {
        p.starts[p.batch] = seen;
        const int left = max(there - pages.b, 0);
        p.free_count_out[0] = left;
        p.free_count_out[1] = static_cast<int>(min(static_cast<int64_t>(pages.b) - (there - left) + static_cast<int64_t>(over), static_cast<int64_t>(0x7fffffff)));
    }
}

// ---- the accepted path ------------------------------------------------------------------------------------
constexpr int kKeepThreads = 128;
constexpr int kAhead = 8;      // rows read before the first of them is written

struct KeepParams {
    uint4 *k, *v;
    const int32_t *tables, *lens, *paths, *held;      // held: nullptr, or the pages that the requests have
    int32_t *lens_out;
    int64_t table_stride, path_stride, layer_stride, page_stride, head_stride, row_stride, num_pages;      // strides of the cache in 16-byte vectors
    int width, page_shift, depth, kv_heads, row_vecs;
};

// CTA -> (request, layer and cache, part of a token's vectors).  A path ascends, so a row that is moved is never one that an earlier move has overwritten.
__global__ void __launch_bounds__(kKeepThreads) keep_kernel(const __grid_constant__ KeepParams p) {
    grid_dependency_sync();
    const int request = blockIdx.x, layer = blockIdx.y >> 1, vec = blockIdx.z * kKeepThreads + threadIdx.x;
    uint4 *cache = (blockIdx.y & 1 ? p.v : p.k) + layer * p.layer_stride;
    const int32_t *path = p.paths + request * p.path_stride, *table = p.tables + request * p.table_stride;
    const int64_t lens = max(p.lens[request], 0), room = static_cast<int64_t>(p.width) << p.page_shift;
    const int64_t bound = p.held ? static_cast<int64_t>(max(p.held[request], 0)) << p.page_shift : INT64_MAX;
    const bool mine = vec < p.kv_heads * p.row_vecs;
    const int64_t inside = mine ? vec / p.row_vecs * p.head_stride + vec % p.row_vecs : 0;
    // nullptr where there is no such row
    auto row_of = [&](int64_t token) -> uint4 * {
        const int64_t at = lens + token;
        if (!mine || at >= room) return nullptr;
        const int32_t id = table[at >> p.page_shift];
        return id < 0 || id >= p.num_pages ? nullptr : cache + id * p.page_stride + (at & ((1 << p.page_shift) - 1)) * p.row_stride + inside;
    };
    int last = -1, count = 0;      // of the path so far
    bool ends = false;
    for (int base = 0; base < p.depth && !ends; base += kAhead) {
        uint4 held[kAhead];
        uint4 *to[kAhead];
        int node[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) node[j] = base + j < p.depth ? path[base + j] : -1;
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            to[j] = nullptr;
            ends = ends || node[j] <= last || lens + node[j] >= bound;      // the path's end, or no path, or a node without a page
            if (ends) continue;
            last = node[j];
            if (node[j] != count) {
                const uint4 *from = row_of(node[j]);
                to[j] = row_of(count);
                if (!from) to[j] = nullptr;
                else if (to[j]) held[j] = *from;
            }
            ++count;
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            if (to[j]) *to[j] = held[j];
    }
    if (blockIdx.y == 0 && vec == 0) p.lens_out[request] = static_cast<int32_t>(min(lens + count, static_cast<int64_t>(0x7fffffff)));
}

// No trees, those of up to 64 nodes, and larger ones.
const void *plan_of(int words) {
    if (words == 0) return reinterpret_cast<const void *>(&plan_kernel<0>);
    return words <= 2 ? reinterpret_cast<const void *>(&plan_kernel<2>) : reinterpret_cast<const void *>(&plan_kernel<kMaxWords>);
}
int page_shift_of(int page_size) {
    int s = 0;
    while ((1 << s) < page_size) ++s;
    return s;
}
bool power_of_two(int v) { return v > 0 && (v & (v - 1)) == 0; }

}  // namespace

cudaError_t paged_ops_setup(DecodeDevice *d) {
    cudaError_t e = cudaSuccess;
    d->plan_ctas = kPlanCtas;
    for (int words : {0, 2, kMaxWords}) {
        if (e == cudaSuccess) e = cudaFuncSetAttribute(plan_of(words), cudaFuncAttributeMaxDynamicSharedMemorySize, (5 * kMaxRequests + 1) * 4);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(plan_of(words), cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        while (e == cudaSuccess && d->plan_ctas > 1) {
            int64_t ctas = 0;
            if (resident_ctas(plan_of(words), kPlanThreads, d->plan_ctas, d->sms, &ctas, (5 * kMaxRequests + 1) * 4) != cudaSuccess) cudaGetLastError(), ctas = 0;
            if (ctas >= d->plan_ctas) break;
            d->plan_ctas /= 2;
        }
    }
    return e;
}

}  // namespace gpuk

int gpuk::paged_plan_ctas_tuning = 0;

using namespace gpuk;

extern "C" int gpuk_paged_plan(const int32_t *lens, const int32_t *new_lens, int32_t *tables, int64_t table_stride, int table_width, const int32_t *held, int32_t *free_pages,
                               int free_capacity, const int32_t *free_count, const int32_t *parents, int batch, int total, int page_size, int mask_words, int32_t *starts,
                               int64_t *positions, int64_t *slots, int32_t *masks, int32_t *held_out, int32_t *free_count_out, void *stream) {
    if (batch < 0 || total < 0 || table_width < 0 || table_stride < 0 || free_capacity < 0 || mask_words < 0)
        return set_last_error(GPUK_ERR_INVALID_ARGUMENT, "paged_plan: bad sizes");
    if (!power_of_two(page_size) || page_size > 65536) return set_last_error(GPUK_ERR_UNSUPPORTED, "paged_plan: pages of %d tokens; built for powers of two up to 65536", page_size);
    if (batch > kMaxRequests) return set_last_error(GPUK_ERR_UNSUPPORTED, "paged_plan: %d requests; built for at most %d", batch, kMaxRequests);
    if (total == 0) parents = nullptr, masks = nullptr;      // of no tokens there may be neither, or only an address
    if (!parents != !masks || (masks && (mask_words < 1 || mask_words > kMaxWords)))
        return set_last_error(GPUK_ERR_INVALID_ARGUMENT, "paged_plan: parents come with masks of 1 to %d words", kMaxWords);
    if (static_cast<int64_t>(batch) * table_width > 0x7fffffffll || static_cast<int64_t>(table_width) * page_size > 0x7fffff00ll)
        return set_last_error(GPUK_ERR_UNSUPPORTED, "paged_plan: tables of %d x %d pages are too large", batch, table_width);
    if (!starts || !free_count || !free_count_out || (batch && (!lens || !new_lens || !held || !held_out || (table_width && !tables))) || (free_capacity && !free_pages) ||
        (total && (!positions || !slots)))
        return set_last_error(GPUK_ERR_INVALID_ARGUMENT, "paged_plan: null pointer");
    if (total > kCeiling) return set_last_error(GPUK_ERR_UNSUPPORTED, "paged_plan: %d tokens are too many", total);
    const DecodeDevice *d = nullptr;
    const int rc = decode_device(&d);
    if (rc != GPUK_OK) return rc;
    PlanParams p = {lens, new_lens, held, free_count, parents, tables, free_pages, starts, masks, held_out, free_count_out, positions, slots, table_stride, batch, table_width,
                    page_shift_of(page_size), free_capacity, total, mask_words};
    int ctas = 1;
    const int most = paged_plan_ctas_tuning && paged_plan_ctas_tuning < d->plan_ctas ? paged_plan_ctas_tuning : d->plan_ctas;
    while (ctas < most && total > ctas * kPlanThreads) ctas *= 2;
    void *args[] = {&p};
    const cudaError_t e = launch_kernel(plan_of(masks ? mask_words : 0), ctas, kPlanThreads, ctas, false, args, static_cast<cudaStream_t>(stream), (5 * batch + 1) * 4);
    if (e != cudaSuccess) return set_last_error(GPUK_ERR_CUDA, "paged_plan: launch failed: %s", cudaGetErrorString(e));
    return GPUK_OK;
}

extern "C" int gpuk_paged_keep(const gpuk_pages *pages, int layers, int64_t layer_stride, const int32_t *tables, int64_t table_stride, int table_width, const int32_t *lens,
                               const int32_t *paths, int64_t path_stride, int depth, int32_t *lens_out, int batch, void *stream) {
    return gpuk_paged_keep_held(pages, layers, layer_stride, tables, table_stride, table_width, lens, paths, path_stride, depth, nullptr, lens_out, batch, stream);
}

extern "C" int gpuk_paged_keep_held(const gpuk_pages *pages, int layers, int64_t layer_stride, const int32_t *tables, int64_t table_stride, int table_width, const int32_t *lens,
                                    const int32_t *paths, int64_t path_stride, int depth, const int32_t *held, int32_t *lens_out, int batch, void *stream) {
    if (!pages) return set_last_error(GPUK_ERR_INVALID_ARGUMENT, "paged_keep: no pages");
    if (batch < 0 || layers <= 0 || depth < 0 || table_width < 0 || pages->kv_heads <= 0 || pages->head_dim <= 0 || pages->num_pages < 0)
        return set_last_error(GPUK_ERR_INVALID_ARGUMENT, "paged_keep: bad sizes");
    if (pages->dtype != GPUK_DTYPE_BF16 && pages->dtype != GPUK_DTYPE_F16) return set_last_error(GPUK_ERR_UNSUPPORTED, "paged_keep: built for bf16 and fp16");
    if (pages->head_dim % 8 || static_cast<int64_t>(pages->kv_heads) * pages->head_dim > 1 << 24)
        return set_last_error(GPUK_ERR_UNSUPPORTED, "paged_keep: heads of %d are no multiple of 8, or too many", pages->head_dim);
    if (!power_of_two(pages->page_size) || pages->page_size > 65536) return set_last_error(GPUK_ERR_UNSUPPORTED, "paged_keep: pages of %d tokens; built for powers of two up to 65536", pages->page_size);
    if (layers > 32767) return set_last_error(GPUK_ERR_UNSUPPORTED, "paged_keep: too many layers");
    if (batch == 0) return GPUK_OK;
    if (!lens || !lens_out || (depth && !paths) || (table_width && !tables) || !pages->k || !pages->v) return set_last_error(GPUK_ERR_INVALID_ARGUMENT, "paged_keep: null pointer");
    if ((reinterpret_cast<uintptr_t>(pages->k) | reinterpret_cast<uintptr_t>(pages->v)) & 15u) return set_last_error(GPUK_ERR_INVALID_ARGUMENT, "paged_keep: pointers must be 16-byte aligned");
    for (int64_t s : {layer_stride, pages->page_stride, pages->head_stride, pages->row_stride})
        if (s < 0 || s % 8) return set_last_error(GPUK_ERR_INVALID_ARGUMENT, "paged_keep: strides must be multiples of 8 values");
    KeepParams p = {static_cast<uint4 *>(pages->k), static_cast<uint4 *>(pages->v), tables, lens, paths, held, lens_out, table_stride, path_stride, layer_stride / 8,
                    pages->page_stride / 8, pages->head_stride / 8, pages->row_stride / 8, pages->num_pages, table_width, page_shift_of(pages->page_size), depth, pages->kv_heads,
                    pages->head_dim / 8};
    // the launch below takes three dimensions
    const int64_t parts = (static_cast<int64_t>(p.kv_heads) * p.row_vecs + kKeepThreads - 1) / kKeepThreads;
    if (parts > 65535) return set_last_error(GPUK_ERR_UNSUPPORTED, "paged_keep: too many heads");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(batch, 2 * layers, static_cast<unsigned>(parts));
    cfg.blockDim = dim3(kKeepThreads);
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    void *args[] = {&p};
    const cudaError_t e = cudaLaunchKernelExC(&cfg, reinterpret_cast<const void *>(&keep_kernel), args);
    if (e != cudaSuccess) return set_last_error(GPUK_ERR_CUDA, "paged_keep: launch failed: %s", cudaGetErrorString(e));
    return GPUK_OK;
}
