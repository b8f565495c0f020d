// Rotary embedding of heads in any of the three orders of pairs, of the whole head or its first `rotary` values, with the keys and values going to their slots of a
// paged cache or a single tensor rotated by itself.
//
// Angles are not read from a table but computed: a frequency is given in turns a position, as a fixed-point fraction of 64 bits, so that position * frequency modulo 2^64 is the
// exact fraction of a turn at any position (in fp32 the angle of position 2^20 would be off by 0.06), and sincospi of its upper bits has no large argument to reduce.
// A CTA works on one token: it computes the rotary / 2 sines and cosines once, into shared memory, while its loads are in flight, and uses them for all its heads.
//
// Bound by HBM for prompts, where a token is 2 * (heads + 2 kv_heads) * head_dim values of traffic, and by latency for a decode step, where a token's heads are dealt
// out to several CTAs.  fp32 products and sums, one rounding; what is not rotated is copied bit for bit.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/gpuk_b200.h"
#include "common.cuh"
#include "launch.cuh"
#include "linear.cuh"

namespace gpuk {
namespace {

constexpr int kVec = 16;          // values an item covers: eight pairs, or two vectors that are copied
constexpr int kItems = 2;         // of a thread, loaded before the first is used
constexpr int kMaxRotary = 256;

struct RopeSource {
    const void *x;
    int64_t token, head;          // strides in values
};
struct RopeParams {
    RopeSource q, k, v;           // k and v: nullptr without a cache
    void *q_out;
    int64_t out_token, out_head;
    void *k_pages, *v_pages;
    int64_t page_stride, head_stride, row_stride, num_pages;
    const int64_t *positions, *slots, *turns;      // turns a position, fractions of 2^64
    float amplitude;
    int tokens, heads, kv_heads, head_dim, rotary, page_shift, layout;
    int chunks, chunk_items;      // CTAs a token, items of each
    int streaming;                // more is written than L2 keeps until it is read
    int *status;
};

template <typename T>
__global__ void rope_kernel(const __grid_constant__ RopeParams p) {
    __shared__ float2 angles[kMaxRotary / 2];
    grid_dependency_sync();
    const int token = blockIdx.x / p.chunks, chunk = blockIdx.x - token * p.chunks;
    const int parts = p.head_dim / kVec, turned = p.rotary / kVec, half = p.rotary / 2;
    const int all = (p.k.x ? p.heads + 2 * p.kv_heads : p.heads) * parts;
    const int first = chunk * p.chunk_items, end = min(first + p.chunk_items, all);
    const bool paged = p.slots != nullptr;
    const int64_t position = p.positions[token], slot = paged ? p.slots[token] : 0;
    const bool there = slot >= 0 && (!paged || slot >> p.page_shift < p.num_pages);

    // an item is at `a` and, its second half, at `b` of its head, and goes to `c` and `d`
    uint4 in[kItems][2];
    const T *src[kItems];
    int head[kItems], a[kItems], b[kItems], pair[kItems];
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
        const int item = first + i * blockDim.x + threadIdx.x;
        head[i] = -1;
        if (item >= end) continue;
        const int h = item / parts, part = item - h * parts, kv = h - p.heads;
        const bool rotated = part < turned && kv < p.kv_heads;
        const RopeSource &s = kv < 0 ? p.q : kv < p.kv_heads ? p.k : p.v;
        const int local = kv < 0 ? h : kv < p.kv_heads ? kv : kv - p.kv_heads;
        head[i] = h;
        pair[i] = rotated ? part * (kVec / 2) : -1;
        const bool halves = rotated && p.layout == GPUK_ROPE_HALF;
        a[i] = halves ? part * (kVec / 2) : part * kVec;
        b[i] = halves ? half + a[i] : a[i] + kVec / 2;
        src[i] = static_cast<const T *>(s.x) + token * s.token + local * s.head;
        in[i][0] = ld_stream(reinterpret_cast<const uint4 *>(src[i] + a[i]));
        in[i][1] = ld_stream(reinterpret_cast<const uint4 *>(src[i] + b[i]));
    }
    for (int i = threadIdx.x; i < half; i += blockDim.x) {
        const uint64_t turn = static_cast<uint64_t>(position) * static_cast<uint64_t>(p.turns[i]);
        float s, c;
        sincospif(static_cast<float>(static_cast<int32_t>(turn >> 32)) * 0x1p-31f, &s, &c);      // the turn from -1/2 to 1/2, in units of half a turn
        angles[i] = make_float2(c * p.amplitude, s * p.amplitude);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
        if (head[i] < 0) continue;
        const int kv = head[i] - p.heads;
        uint4 lo = in[i][0], hi = in[i][1];
        int c = a[i], d = b[i];
        if (pair[i] >= 0) {
            float x[16], y[16];
            Elem<T>::unpack(lo, *reinterpret_cast<float(*)[8]>(x));
            Elem<T>::unpack(hi, *reinterpret_cast<float(*)[8]>(x + 8));
            if (p.layout == GPUK_ROPE_HALF) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float2 t = angles[pair[i] + e];
                    y[e] = x[e] * t.x - x[8 + e] * t.y;
                    y[8 + e] = x[8 + e] * t.x + x[e] * t.y;
                }
            } else {
                float u[8], w[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float2 t = angles[pair[i] + e];
                    u[e] = x[2 * e] * t.x - x[2 * e + 1] * t.y;
                    w[e] = x[2 * e + 1] * t.x + x[2 * e] * t.y;
                }
                const bool split = p.layout == GPUK_ROPE_SPLIT;
                if (split) c = pair[i], d = half + pair[i];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    y[e] = split ? u[e] : e & 1 ? w[e / 2] : u[e / 2];
                    y[8 + e] = split ? w[e] : e & 1 ? w[4 + e / 2] : u[4 + e / 2];
                }
            }
            lo = Elem<T>::pack(*reinterpret_cast<float(*)[8]>(y));
            hi = Elem<T>::pack(*reinterpret_cast<float(*)[8]>(y + 8));
        }
        T *dst;
        if (kv < 0) {
            dst = static_cast<T *>(p.q_out) + token * p.out_token + head[i] * p.out_head;
            // a token without a place is marked: its keys are nowhere
            if (!there) lo = hi = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
        } else {
            if (!there) continue;
            const bool key = kv < p.kv_heads;
            dst = static_cast<T *>(key ? p.k_pages : p.v_pages) + (slot >> p.page_shift) * p.page_stride + (key ? kv : kv - p.kv_heads) * p.head_stride +
                  (slot & ((1 << p.page_shift) - 1)) * p.row_stride;
        }
        if (p.streaming) {
            __stcs(reinterpret_cast<uint4 *>(dst + c), lo);
            __stcs(reinterpret_cast<uint4 *>(dst + d), hi);
        } else {
            *reinterpret_cast<uint4 *>(dst + c) = lo;
            *reinterpret_cast<uint4 *>(dst + d) = hi;
        }
    }
    if (!there && slot >= 0 && threadIdx.x == 0) *p.status = 1;
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool bad_stride(int64_t s) { return s < 0 || s % 8; }

int launch(RopeParams &p, int dtype, void *stream, const char *what) {
    if (dtype != GPUK_DTYPE_BF16 && dtype != GPUK_DTYPE_F16) return set_last_error(GPUK_ERR_UNSUPPORTED, "%s: built for bf16 and fp16", what);
    if (p.tokens < 0 || p.heads < 0 || p.kv_heads < 0 || p.head_dim <= 0 || p.heads + p.kv_heads == 0) return set_last_error(GPUK_ERR_INVALID_ARGUMENT, "%s: bad sizes", what);
    if (p.head_dim % kVec || p.rotary % kVec || p.rotary <= 0 || p.rotary > p.head_dim || p.rotary > kMaxRotary)
        return set_last_error(GPUK_ERR_UNSUPPORTED, "%s: heads of %d, %d of it rotated; built for multiples of %d, at most %d rotated", what, p.head_dim, p.rotary, kVec, kMaxRotary);
    if (p.layout < GPUK_ROPE_HALF || p.layout > GPUK_ROPE_SPLIT) return set_last_error(GPUK_ERR_INVALID_ARGUMENT, "%s: unknown layout %d", what, p.layout);
    const int64_t items = (p.heads + 2ll * p.kv_heads) * (p.head_dim / kVec);
    if (items > 1 << 24) return set_last_error(GPUK_ERR_UNSUPPORTED, "%s: too many heads", what);
    if (p.tokens == 0) return GPUK_OK;
    if (!p.positions || !p.turns) return set_last_error(GPUK_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
    const DecodeDevice *d = nullptr;
    const int rc = decode_device(&d);
    if (rc != GPUK_OK) return rc;
    p.status = d->status + kStatusPosition;
    // few tokens: more CTAs for each, so that there are two for each SM; else the fewest of at most 256 threads
    const int least = static_cast<int>((items + 256 * kItems - 1) / (256 * kItems));
    int64_t chunks = (2ll * d->sms + p.tokens - 1) / p.tokens;
    if (chunks * 64 > items) chunks = (items + 63) / 64;
    if (chunks < least) chunks = least;
    p.chunk_items = static_cast<int>((items + chunks - 1) / chunks);
    p.chunks = static_cast<int>((items + p.chunk_items - 1) / p.chunk_items);
    // 8191 tokens of 64 + 16 heads of 128: 59.4 us, 62.5 with stores that stay in L2; a step of a few tokens is read from there by the attention behind it
    p.streaming = p.tokens * items * (kVec * 2) > 64ll << 20;
    const int threads = (p.chunk_items + kItems - 1) / kItems;
    if (static_cast<int64_t>(p.tokens) * p.chunks > 0x7fffffffll) return set_last_error(GPUK_ERR_UNSUPPORTED, "%s: too many tokens", what);
    const void *fn = dtype == GPUK_DTYPE_BF16 ? reinterpret_cast<const void *>(&rope_kernel<__nv_bfloat16>) : reinterpret_cast<const void *>(&rope_kernel<__half>);
    void *args[] = {&p};
    const cudaError_t e = launch_kernel(fn, p.tokens * p.chunks, (threads + 31) / 32 * 32, 1, false, args, static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) return set_last_error(GPUK_ERR_CUDA, "%s: launch failed: %s", what, cudaGetErrorString(e));
    return GPUK_OK;
}

}  // namespace
}  // namespace gpuk

using namespace gpuk;

extern "C" int gpuk_rope(const void *x, int64_t token_stride, int64_t head_stride, void *out, int64_t out_token_stride, int64_t out_head_stride, const int64_t *positions,
                         const int64_t *turns, float amplitude, int tokens, int heads, int head_dim, int rotary, int layout, int dtype, void *stream) {
    if (tokens > 0 && heads > 0 && (!x || !out || !aligned16(x) || !aligned16(out)))
        return set_last_error(GPUK_ERR_INVALID_ARGUMENT, "rope: pointers must be 16-byte aligned and not null");
    for (int64_t s : {token_stride, head_stride, out_token_stride, out_head_stride})
        if (bad_stride(s)) return set_last_error(GPUK_ERR_INVALID_ARGUMENT, "rope: strides must be multiples of 8 values");
    RopeParams p = {};
    p.q = {x, token_stride, head_stride};
    p.q_out = out, p.out_token = out_token_stride, p.out_head = out_head_stride;
    p.positions = positions, p.turns = turns, p.amplitude = amplitude;
    p.tokens = tokens, p.heads = heads, p.head_dim = head_dim, p.rotary = rotary, p.layout = layout;
    return launch(p, dtype, stream, "rope");
}

extern "C" int gpuk_rope_paged(const void *q, int64_t q_token_stride, int64_t q_head_stride, const void *k, int64_t k_token_stride, int64_t k_head_stride, const void *v,
                               int64_t v_token_stride, int64_t v_head_stride, void *q_out, int64_t out_token_stride, int64_t out_head_stride, const int64_t *positions,
                               const int64_t *slots, const int64_t *turns, float amplitude, const gpuk_pages *pages, int tokens, int heads, int rotary, int layout, void *stream) {
    if (!pages) return set_last_error(GPUK_ERR_INVALID_ARGUMENT, "rope_paged: no pages");
    if (pages->kv_heads <= 0 || pages->num_pages < 0) return set_last_error(GPUK_ERR_INVALID_ARGUMENT, "rope_paged: bad sizes");
    const int size = pages->page_size;
    if (size <= 0 || (size & (size - 1)) || size > 65536) return set_last_error(GPUK_ERR_UNSUPPORTED, "rope_paged: pages of %d tokens; built for powers of two up to 65536", size);
    if (tokens > 0) {
        for (const void *x : {static_cast<const void *>(pages->k), static_cast<const void *>(pages->v), k, v, static_cast<const void *>(slots)})
            if (!x) return set_last_error(GPUK_ERR_INVALID_ARGUMENT, "rope_paged: null pointer");
        if (heads > 0 && (!q || !q_out)) return set_last_error(GPUK_ERR_INVALID_ARGUMENT, "rope_paged: null pointer");
        for (const void *x : {static_cast<const void *>(pages->k), static_cast<const void *>(pages->v), k, v, q, static_cast<const void *>(q_out)})
            if (!aligned16(x)) return set_last_error(GPUK_ERR_INVALID_ARGUMENT, "rope_paged: pointers must be 16-byte aligned");
    }
    for (int64_t s : {q_token_stride, q_head_stride, k_token_stride, k_head_stride, v_token_stride, v_head_stride, out_token_stride, out_head_stride, pages->page_stride,
                      pages->head_stride, pages->row_stride})
        if (bad_stride(s)) return set_last_error(GPUK_ERR_INVALID_ARGUMENT, "rope_paged: strides must be multiples of 8 values");
    RopeParams p = {};
    p.q = {q, q_token_stride, q_head_stride}, p.k = {k, k_token_stride, k_head_stride}, p.v = {v, v_token_stride, v_head_stride};
    p.q_out = q_out, p.out_token = out_token_stride, p.out_head = out_head_stride;
    p.k_pages = pages->k, p.v_pages = pages->v;
    p.page_stride = pages->page_stride, p.head_stride = pages->head_stride, p.row_stride = pages->row_stride, p.num_pages = pages->num_pages;
    p.positions = positions, p.slots = slots, p.turns = turns, p.amplitude = amplitude;
    p.tokens = tokens, p.heads = heads, p.kv_heads = pages->kv_heads, p.head_dim = pages->head_dim, p.rotary = rotary, p.layout = layout;
    while ((1 << p.page_shift) < size) ++p.page_shift;
    return launch(p, pages->dtype, stream, "rope_paged");
}
