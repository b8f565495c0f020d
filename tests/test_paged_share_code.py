"""The shares of the paged attention kernels, by their own code: ``csrc/paged_share.cuh`` compiled for the host, a warp's lanes as fibers that meet at its shuffles.

Every block of every tile is taken once, in order, and the second kernel's search finds each part in the slot that it was left in.  Quotients and roots that the device only estimates are off
by a few units here, in either direction at random, as its approximations may be."""
import ctypes
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUDA = os.environ.get("CUDA_HOME", "/usr/local/cuda")

HARNESS = r"""
#include <cuda_runtime.h>
#include <ucontext.h>
#include <cmath>
#include <cstdint>
#include <vector>

static struct { unsigned x; } threadIdx, blockIdx, gridDim;
template <typename T> static T min(T a, T b) { return a < b ? a : b; }
template <typename T> static T max(T a, T b) { return a < b ? b : a; }
static float __uint_as_float(unsigned) { return 0.f; }      // not called
static unsigned __umulhi(unsigned a, unsigned b) { return static_cast<unsigned>((static_cast<uint64_t>(a) * b) >> 32); }

static uint64_t noise_state = 1;
static float off(float x) {
    noise_state = noise_state * 6364136223846793005ull + 1442695040888963407ull;
    return x * (1.f + static_cast<float>(static_cast<int>(noise_state >> 40 & 7) - 3) * 0x1p-22f);
}
static float __fdividef(float a, float b) { return off(a / b); }
static float estimated_root(float x) { return off(std::sqrt(x)); }
#define sqrtf estimated_root

// Lanes run in turn, each up to its next meeting; what they bring there lies in one of two rows, so that a lane that is ahead overwrites nothing.
static ucontext_t lanes[32], home;
static int64_t brought[2][32];
static int meetings[32], current;
static bool over[32];
static std::vector<char> stacks[32];
static int64_t *meet(int64_t v) {
    const int me = current, row = meetings[me]++ & 1;
    brought[row][me] = v;
    swapcontext(&lanes[me], &home);
    return brought[row];
}
template <typename T> static T __shfl_up_sync(unsigned, T v, int o) { const int me = current; int64_t *r = meet(v); return static_cast<T>(r[me >= o ? me - o : me]); }
template <typename T> static T __shfl_sync(unsigned, T v, int lane) { return static_cast<T>(meet(v)[lane]); }
static int __reduce_add_sync(unsigned, int v) { int64_t *r = meet(v), s = 0; for (int i = 0; i < 32; ++i) s += r[i]; return static_cast<int>(s); }
static unsigned __reduce_max_sync(unsigned, unsigned v) { int64_t *r = meet(v), s = 0; for (int i = 0; i < 32; ++i) s = r[i] > s ? r[i] : s; return static_cast<unsigned>(s); }
static void __syncwarp() { meet(0); }

#include "paged_share.cuh"

using namespace gpuk;
static const PagedAttentionParams *params;
static Start *place;
static int border_side;
static void lane_main() {
    find_border(*params, place, border_side);
    over[current] = true;
    swapcontext(&lanes[current], &home);
}
static void warp(const PagedAttentionParams &p, Start *out, int side) {
    params = &p, place = out, border_side = side;
    for (int i = 0; i < 32; ++i) {
        stacks[i].resize(64 << 10);
        getcontext(&lanes[i]);
        lanes[i].uc_stack.ss_sp = stacks[i].data(), lanes[i].uc_stack.ss_size = stacks[i].size(), lanes[i].uc_link = nullptr;
        makecontext(&lanes[i], lane_main, 0);
        meetings[i] = 0, over[i] = false;
    }
    for (bool going = true; going;) {
        going = false;
        for (int i = 0; i < 32; ++i) {
            if (over[i]) continue;
            going = true, current = i, threadIdx.x = i;
            swapcontext(&home, &lanes[i]);
        }
    }
}

// Segments of each CTA: ten numbers each (cta, request, kv head, first token, first block, blocks, all blocks of the tile, slot, begins, ends).  Returns their number; ctas: those that take part.
extern "C" int shares(int batch, int tokens, const int *starts, const int *lens, int masks, int kv_heads, int tile_tokens, int width, int page_shift, int may_split, int grid, uint64_t seed,
                      int64_t *out, int most, int *ctas) {
    PagedAttentionParams p = {};
    p.starts = starts, p.lens = lens, p.masks = masks ? starts : nullptr;
    p.batch = batch, p.tokens = tokens, p.kv_heads = kv_heads, p.tile_tokens = tile_tokens;
    p.tile_inverse = static_cast<uint32_t>(((1ull << 32) + tile_tokens - 1) / tile_tokens);
    p.width = width, p.page_shift = page_shift, p.may_split = may_split;
    gridDim.x = grid, noise_state = seed;
    int n = 0;
    for (int c = 0; c < grid; ++c) {
        blockIdx.x = c;
        Start s = {};
        warp(p, &s, 0), warp(p, &s, 1);
        *ctas = s.ctas;
        if (s.x[1] <= s.x[0]) continue;
        Walk walk(s);
        Segment u;
        bool begins, ends;
        while (walk.next(p, &u, &begins, &ends)) {
            if (n == most) return -1;
            const int64_t all = (keys_of(p, walk.r, u.tok0 / tile_tokens) + kKeys - 1) / kKeys;
            const int64_t row[10] = {c, u.request, u.kvh, u.tok0, u.first, u.blocks, all, u.slot, begins, ends};
            for (int i = 0; i < 10; ++i) out[n * 10 + i] = row[i];
            ++n;
        }
    }
    return n;
}
extern "C" void constants(int *out) { out[0] = kKeys, out[1] = kTileCost, out[2] = kFront, out[3] = kGrain, out[4] = kPerCta, out[5] = kSmall; }
"""


@pytest.fixture(scope="module")
def code(tmp_path_factory):
    folder = tmp_path_factory.mktemp("share")
    (folder / "share.cpp").write_text(HARNESS)
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-w", "-I", os.path.join(CUDA, "include"), "-I", os.path.join(ROOT, "gpuk_b200", "csrc"), "-o", str(folder / "share.so"),
                    str(folder / "share.cpp")], check=True)
    return ctypes.CDLL(str(folder / "share.so"))


def _ints(values):
    return (ctypes.c_int * max(1, len(values)))(*values)


def _check(code, requests, kv, tile_tokens, masks, width, page_shift, split, grid, seed, spare=0):
    """`requests`: cached and new tokens; those behind `spare` rows of q are there too."""
    starts = [sum(n for _, n in requests[:i]) for i in range(len(requests) + 1)]
    most, ctas = 400000, ctypes.c_int()
    out = (ctypes.c_int64 * (10 * most))()
    count = code.shares(len(requests), starts[-1] + spare, _ints(starts), _ints([c for c, _ in requests]), masks, kv, tile_tokens, width, page_shift, split, grid, ctypes.c_uint64(seed), out, most,
                        ctypes.byref(ctas))
    assert count >= 0 and 1 <= ctas.value <= grid
    taken, slots, of = {}, {}, {}
    for i in range(count):
        c, request, kvh, tok0, first, blocks, every, slot, begins, ends = out[10 * i:10 * i + 10]
        assert c < ctas.value and 0 <= first and blocks > 0 and first + blocks <= every
        tile = (request, kvh, tok0)
        taken.setdefault(tile, []).append((first, first + blocks, every))
        of.setdefault(c, []).append((tile, slot, begins, ends))
        assert (slot < 0) == bool(begins and ends)
        if slot >= 0:
            assert slot // 2 == c and slot not in slots and split
            slots[slot] = tile
    want = {(i, h, t) for i, (_, n) in enumerate(requests) for h in range(kv) for t in range(0, n, tile_tokens)}
    assert set(taken) == want
    room = width << page_shift
    for (i, _, t), pieces in taken.items():
        c, n = requests[i]
        keys = min(min(max(c, 0), room) + (n if masks else min(n, t + tile_tokens)), room)
        assert pieces[0][0] == 0 and pieces[-1][1] == pieces[-1][2] == -(-keys // 64) and all(a[1] == b[0] for a, b in zip(pieces, pieces[1:]))
    # what the second kernel does: from the CTA where a tile begins to the one where it ends
    head = [0] * ctas.value
    for c, mine in of.items():
        head[c] = 3 if mine[0][2] else 2 if mine[0][3] else 1
        assert all(begins for _, _, begins, _ in mine[1:]) and all(ends for _, _, _, ends in mine[:-1])
    joined = []
    for c, mine in of.items():
        tile, slot, begins, ends = mine[-1]
        if begins and not ends:
            parts = [slot]
            for d in range(c + 1, ctas.value):
                if head[d] in (1, 2):
                    parts.append(2 * d)
                if head[d] >= 2:
                    break
            assert all(slots.get(s) == tile for s in parts)
            joined += parts
    assert sorted(joined) == sorted(slots)
    return count, len(slots)


@pytest.mark.parametrize("masks", [False, True])
def test_every_block_is_taken_once_and_found_again(code, masks):
    rng, parts = random.Random(masks), 0
    for seed in range(60):
        batch, kv, tt = rng.choice([1, 2, 5, 40, 97]), rng.choice([1, 3, 8]), rng.choice([1, 16, 25, 128])
        longest = rng.choice([10, 400, 3000, 20000])
        requests = [(rng.choice([0, rng.randint(0, longest)]), rng.choice([0, 1, 1, rng.randint(0, 70), rng.randint(0, 300)])) for _ in range(batch)]
        shift = rng.choice([3, 4, 6])
        room = rng.choice([1 << 20, 1 << 20, longest // 2 + 8])
        parts += _check(code, requests, kv, tt, masks, -(-room >> shift), shift, rng.random() < 0.9, rng.choice([1, 7, 64, 296]), seed, rng.choice([0, 5]))[1]
    assert parts > 500


def test_long_contexts_and_many_requests(code):
    """Where an estimate in 32 bits is off by whole blocks and has to be put right: contexts of 2^30 keys, prompts of 2^20 tokens, 4096 requests."""
    rng = random.Random(3)
    _check(code, [(1 << 30, 1), (0, 3), ((1 << 30) - 12345, 130)], 2, 16, False, 1 << 24, 6, True, 296, 1)
    _check(code, [(777, 1 << 18), (0, 1), (5, 4097)], 1, 128, False, 1 << 20, 6, True, 296, 2)
    _check(code, [(rng.randint(0, 3000), rng.choice([0, 1, 1, 1, 40])) for _ in range(4096)], 1, 16, False, 1 << 8, 4, True, 148, 3)
    _check(code, [(0, 0)] * 50, 4, 16, True, 10, 4, True, 296, 4)
    _check(code, [(-5, 3), (2 ** 31 - 1, 20)], 4, 16, True, 10, 4, True, 296, 5)


def test_the_model_has_the_same_numbers(code):
    import tests.test_paged_attention_model as model

    got = (ctypes.c_int * 6)()
    code.constants(got)
    assert list(got) == [model.KEYS, model.COST, model.FRONT, model.GRAIN, model.PER_CTA, model.SMALL]
