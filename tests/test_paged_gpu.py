"""The paged KV cache's operators against plain implementations in 64 bits or whole numbers: plans, rotary positions, attention, accepted paths, and a step of them together."""
import math
import random

import pytest
import torch

import gpuk_b200 as gpuk
from gpuk_b200 import cabi

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
HALF_STEP = {BF16: 2.0 ** -8, F16: 2.0 ** -11}


def _status_ok():
    cabi.check(cabi.lib.gpuk_fp8_linear_status())


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ---- plans -----------------------------------------------------------------------------------------------
def _plain_plan(lens, new, tables, held, free, count, page, total, parents):
    """The plan in Python's whole numbers; lists are changed in place as the call changes them."""
    width, starts, at = len(tables[0]) if tables else 0, [0], 0
    lens, held = [max(c, 0) for c in lens], [min(max(h, 0), width) for h in held]
    fit = []
    for n in new:
        fit.append(min(max(n, 0), total - at))
        at += fit[-1]
        starts.append(at)
    pages = [-(-(c + n) // page) for c, n in zip(lens, fit)]
    need = [min(p, width) for p in pages]
    for i, h in enumerate(held):
        for j in range(need[i], h):
            if count < len(free):
                free[count] = tables[i][j]
            count = min(count + 1, len(free))
    missing, out_held = sum(p - n for p, n in zip(pages, need)), []
    for i, h in enumerate(held):
        got = min(h, need[i])
        for j in range(h, need[i]):
            if count:
                count -= 1
                tables[i][j] = free[count]
                got += 1
            else:
                tables[i][j] = -1
                missing += 1
        out_held.append(got)
    positions, slots, masks = [-1] * total, [-1] * total, [0] * total
    for i, (c, n) in enumerate(zip(lens, fit)):
        seen = []
        for j in range(n):
            t, block = starts[i] + j, (c + j) // page
            if block < width and tables[i][block] >= 0:
                slots[t] = tables[i][block] * page + (c + j) % page
            up = parents[t] if parents else j - 1
            seen.append((seen[up] if 0 <= up < j else 0) | 1 << j)
            positions[t] = c + (bin(seen[j]).count("1") - 1 if parents else j)
            masks[t] = seen[j]
    return starts, positions, slots, masks, out_held, [count, missing]


def _check_plan(lens, new, tables, held, free, count, page, total, parents=None, max_new=0, in_place=False):
    args = [_ints(lens), _ints(new), _ints(tables).view(len(lens), -1), _ints(held), _ints(free), _ints([count, 0])]
    more = {"held_out": args[3], "free_count_out": args[5]} if in_place else {}
    want_tables, want_free = [list(r) for r in tables], list(free)
    starts, positions, slots, masks, want_held, want_count = _plain_plan(lens, new, want_tables, held, want_free, count, page, total, parents)
    for _ in range(1 if in_place else 2):      # the second time with the same arguments
        p = gpuk.paged_plan(*args, page, total, parents=None if parents is None else _ints(parents), max_new=max_new, **more)
        assert p.starts.tolist() == starts
        assert p.positions.tolist() == positions
        assert p.slots.tolist() == slots
        assert p.held.tolist() == want_held
        assert p.free_count.tolist() == want_count
        assert args[2].tolist() == want_tables
        assert args[4].tolist() == want_free
        if parents is not None:
            words = (max_new + 31) // 32
            got = [sum((w & 0xffffffff) << 32 * k for k, w in enumerate(row)) for row in p.masks.tolist()]
            assert got == [m & (1 << 32 * words) - 1 for m in masks]
    if in_place:
        assert p.held.data_ptr() == args[3].data_ptr() and p.free_count.data_ptr() == args[5].data_ptr()


def _random_state(rng, batch, page, ctx, new, spare, slack=0):
    lens, fresh = [rng.randint(0, ctx) for _ in range(batch)], [rng.randint(0, new) for _ in range(batch)]
    width = -(-(ctx + new) // page) + 1
    held = [min(width, -(-c // page) + rng.choice([0, 0, 1, 2])) for c in lens]
    pages = sum(held) + spare
    order = list(range(pages))
    rng.shuffle(order)
    tables, at = [], 0
    for h in held:
        tables.append(order[at:at + h] + [-1] * (width - h))
        at += h
    return lens, fresh, tables, held, order[at:] + [0] * at, pages - at, page, sum(fresh) + slack


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("batch,page,ctx,new,spare,slack", [(1, 16, 0, 1, 4, 0), (1, 1, 5, 3, 9, 0), (3, 16, 40, 20, 20, 5), (33, 8, 100, 64, 400, 0), (70, 64, 3000, 1, 200, 3), (7, 16, 50, 2000, 900, 0),
                                                           (1030, 32, 300, 4, 1500, 0), (2, 16, 0, 9000, 1200, 1)])
def test_plan(batch, page, ctx, new, spare, slack, in_place):
    """One request and more than a CTA's threads, one CTA and a cluster of eight, surplus pages that come back, rows behind the last request."""
    _check_plan(*_random_state(random.Random(batch + page), batch, page, ctx, new, spare, slack), in_place=in_place)


@pytest.mark.parametrize("batch,new,max_new", [(1, 1, 1), (5, 8, 8), (40, 32, 32), (40, 33, 33), (9, 64, 64), (3, 256, 256), (4, 64, 30)])
def test_plan_of_trees(batch, new, max_new):
    """Roots in the middle, chains, parents that are none (the token itself, a later one, far off); trees larger than their masks lose the bits that do not fit."""
    rng = random.Random(new)
    state = _random_state(rng, batch, 16, 100, new, 40 + batch * new // 8, 2)
    parents = []
    for n in state[1]:
        parents += [rng.choice([-1, j - 1, rng.randint(-1, max(j - 1, -1)), j, j + 1, -7, 1 << 30]) for j in range(n)]
    _check_plan(*state, parents=parents + [5, -9], max_new=max_new)


def test_plan_of_a_long_chain():
    _check_plan([17], [256], [[3, 4] + [-1] * 18], [2], list(range(5, 30)) + [0] * 5, 25, 16, 256, parents=list(range(-1, 255)), max_new=256)


def test_plan_where_pages_run_out():
    """The list is short, a row of the table is short, and tokens do not fit the rows: what there is goes out in order, the rest is marked."""
    _check_plan([16, 5, 0], [20, 40, 3], [[1, -1, -1], [2, -1, -1], [-1, -1, -1]], [1, 1, 0], [7, 8, 9, 0, 0], 3, 16, 63)
    _check_plan([16, 5, 0], [60, 40, 3], [[1, -1, -1], [2, -1, -1], [-1, -1, -1]], [1, 1, 0], [7, 8, 0, 0, 0], 2, 16, 103)
    _check_plan([16, 5, 0], [20, 40, 3], [[1, -1, -1], [2, -1, -1], [-1, -1, -1]], [1, 1, 0], [7, 8, 9, 0, 0], 3, 16, 30)
    _check_plan([0, 0], [1, 1], [[-1], [-1]], [0, 0], [0], 0, 16, 2)


def test_plan_of_finished_requests_gives_their_pages_to_others():
    _check_plan([0, 30, 0], [0, 40, 17], [[4, 5, 6, 7, -1], [0, 1, -1, -1, -1], [2, 3, -1, -1, -1]], [4, 2, 2], [9] + [0] * 9, 1, 16, 60)


def test_plan_with_odd_lengths():
    """Negative lengths and counts are none, too many held pages are a full row."""
    _check_plan([-3, 2 ** 31 - 1, 4], [-1, 2, 3], [[1, 2], [3, 4], [5, -1]], [9, -2, 1], [8, 6, 0, 0, 0, 0, 0, 0, 0, 0], 2, 16, 7)
    _check_plan([0], [0], [[0, 1]], [2], [7, 7], 9, 16, 0)


def test_plan_of_nothing():
    p = gpuk.paged_plan(_ints([]), _ints([]), _ints([]).view(0, 4), _ints([]), _ints([3, 2]), _ints([2, 0]), 16, 3)
    assert p.starts.tolist() == [0] and p.positions.tolist() == [-1] * 3 and p.slots.tolist() == [-1] * 3 and p.free_count.tolist() == [2, 0]


# ---- rotary positions ------------------------------------------------------------------------------------
def _rotated(x, positions, f, amplitude, layout):
    """In 64 bits, whole turns taken out first; and the largest magnitude in each pair, which bounds what rounding can do."""
    r = 2 * len(f)
    turn = torch.remainder(positions.cpu().double()[:, None] * (f / (2 * math.pi)), 1.0)[:, None] * (2 * math.pi)
    x = x.cpu().double()
    first, second = (list(range(r // 2)), list(range(r // 2, r))) if layout == "half" else (list(range(0, r, 2)), list(range(1, r, 2)))
    a, b = x[..., first], x[..., second]
    y, size = x.clone(), torch.zeros_like(x)
    if layout == "split":
        first, second = list(range(r // 2)), list(range(r // 2, r))
    y[..., first], y[..., second] = amplitude * (a * turn.cos() - b * turn.sin()), amplitude * (b * turn.cos() + a * turn.sin())
    size[..., first] = size[..., second] = amplitude * (a.abs() + b.abs())
    return y, size


def _check_rotated(got, want, size, dtype):
    """One rounding of the result (half a step, doubled where it falls the other way by the fp32 error in front: 2^-21 of the pair allows 2^-22 for the angle's
    24 bits, times pi, and four roundings of 2^-24); fp16's smallest step."""
    bound = want.abs() * HALF_STEP[dtype] * 1.01 + size * 2.0 ** -20 + 2.0 ** -25
    assert bool(((got.cpu().double() - want).abs() <= bound).all())


SCALINGS = [None, {"kind": "linear", "factor": 4.0}, {"kind": "base", "factor": 8.0}, {"kind": "bands", "factor": 8.0, "low": 1.0, "high": 4.0, "original": 8192},
            {"kind": "yarn", "factor": 16.0, "low": 1.0, "high": 32.0, "original": 4096}]


@pytest.mark.parametrize("layout", ["half", "interleaved", "split"])
@pytest.mark.parametrize("tokens,heads,hd,rotary,dtype,far", [(1, 1, 16, 16, BF16, 1), (3, 5, 64, 32, F16, 100), (700, 7, 128, 128, BF16, 2 ** 20), (2, 64, 128, 64, F16, 2 ** 40), (5, 3, 256, 256, BF16, 9),
                                                             (4, 2, 48, 16, F16, 2 ** 62)])
def test_rope(tokens, heads, hd, rotary, dtype, far, layout):
    g = torch.Generator().manual_seed(tokens + hd)
    x = torch.randn(tokens, heads, hd, generator=g).to(dtype).cuda()
    positions = torch.randint(0, far, (tokens,), generator=g).cuda()
    for scaling in SCALINGS[:1] if far > 2 ** 30 else SCALINGS:
        frequencies = gpuk.rope_frequencies(rotary, 500000.0, scaling=scaling, device="cuda")
        got = gpuk.rope(x, positions, frequencies, layout=layout)
        if far <= 2 ** 30:
            want, size = _rotated(x, positions, *gpuk.paged.scaled_frequencies(rotary, 500000.0, scaling), layout)
        else:      # the fixed-point turns in Python's whole numbers: doubles do not hold such angles
            turns = [[(int(p) * (int(t) % 2 ** 64)) % 2 ** 64 / 2 ** 64 for t in frequencies.turns.tolist()] for p in positions.tolist()]
            want, size = (torch.stack(v) for v in zip(*(
                tuple(u[0] for u in _rotated(x[i:i + 1], torch.ones(1), torch.tensor(turns[i], dtype=torch.float64) * 2 * math.pi, 1.0, layout)) for i in range(tokens))))
        _check_rotated(got, want, size, dtype)
        assert torch.equal(got[..., rotary:], x[..., rotary:])
    _status_ok()


def test_frequencies():
    """The plain ones by their formula, each scaling at its ends: pairs that turn often stay, those that turn seldom are divided."""
    f, _ = gpuk.paged.scaled_frequencies(128, 10000.0)
    assert torch.allclose(f, torch.tensor([10000.0 ** (-2 * i / 128) for i in range(64)], dtype=torch.float64), rtol=1e-14)
    for scaling in SCALINGS[3:]:
        g, amplitude = gpuk.paged.scaled_frequencies(128, 10000.0, scaling)
        turns = scaling["original"] * f / (2 * math.pi)
        assert torch.equal(g[turns > 2 * scaling["high"]], f[turns > 2 * scaling["high"]])
        assert torch.allclose(g[turns < scaling["low"] / 2] * scaling["factor"], f[turns < scaling["low"] / 2], rtol=1e-14)
        assert amplitude == (1.0 if scaling["kind"] == "bands" else 0.1 * math.log(16.0) + 1)
    g, _ = gpuk.paged.scaled_frequencies(128, 10000.0, SCALINGS[2])
    assert math.isclose(float(g[0]), 1.0) and math.isclose(float(g[-1]) * 8, float(f[-1]), rel_tol=1e-12)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rope_in_place_and_strided(layout):
    x = torch.randn(9, 11, 64, generator=torch.Generator().manual_seed(1)).to(BF16).cuda()
    positions, frequencies = torch.arange(9, device="cuda") * 1000, gpuk.rope_frequencies(32, device="cuda")
    part = x[:, 2:7]
    want = gpuk.rope(part.contiguous(), positions, frequencies, layout=layout)
    assert torch.equal(gpuk.rope(part, positions, frequencies, layout=layout), want)
    rest = x[:, 7:].clone()
    assert gpuk.rope(part, positions, frequencies, layout=layout, out=part).data_ptr() == part.data_ptr()
    assert torch.equal(x[:, 2:7], want) and torch.equal(x[:, 7:], rest)


def _pool(pages, kv, page, hd, dtype, order="hnd", fill=0.0):
    shape = {"hnd": (pages, kv, page, hd), "nhd": (pages, page, kv, hd), "wide": (pages, kv, page, 2 * hd)}[order]
    t = torch.full(shape, fill, dtype=dtype, device="cuda")
    return t.transpose(1, 2) if order == "nhd" else t[..., :hd] if order == "wide" else t


@pytest.mark.parametrize("order", ["hnd", "nhd", "wide"])
@pytest.mark.parametrize("tokens,heads,kv,hd,rotary,page,dtype,layout", [(1, 8, 1, 128, 128, 16, BF16, "split"), (37, 5, 5, 64, 32, 8, F16, "half"), (300, 28, 4, 128, 64, 1, BF16, "interleaved"),
                                                                        (64, 64, 8, 128, 128, 64, BF16, "half")])
def test_rope_paged(tokens, heads, kv, hd, rotary, page, dtype, layout, order):
    """Queries, keys and values as slices of one projection; every slot that is not written keeps what it held."""
    g = torch.Generator().manual_seed(tokens)
    pages = -(-tokens // page) + 2
    qkv = torch.randn(tokens, heads + 2 * kv, hd, generator=g).to(dtype).cuda()
    q, k, v = qkv.split([heads, kv, kv], dim=1)
    positions = torch.randint(0, 5000, (tokens,), generator=g).cuda()
    slots = torch.randperm(pages * page, generator=g)[:tokens].cuda()
    frequencies = gpuk.rope_frequencies(rotary, 10000.0, device="cuda")
    f, amplitude = gpuk.paged.scaled_frequencies(rotary, 10000.0)
    kc, vc = _pool(pages, kv, page, hd, dtype, order, 7.0), _pool(pages, kv, page, hd, dtype, order, 9.0)
    got = gpuk.rope_paged(q, k, v, positions, slots, frequencies, kc, vc, layout=layout)
    _status_ok()
    _check_rotated(got, *_rotated(q, positions, f, amplitude, layout), dtype)
    assert torch.equal(got, gpuk.rope(q, positions, frequencies, layout=layout))
    flat_k, flat_v = (c.transpose(1, 2).reshape(pages * page, kv, hd) for c in (kc, vc))
    assert torch.equal(flat_k[slots], gpuk.rope(k, positions, frequencies, layout=layout)) and torch.equal(flat_v[slots], v)
    rest = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    rest[slots] = False
    assert bool((flat_k[rest] == 7).all()) and bool((flat_v[rest] == 9).all())


def test_rope_paged_without_a_place():
    """A token with no slot, or one behind the last, writes nothing; its queries are marked; only the latter is an error."""
    x = torch.ones(4, 3, 16, device="cuda").to(BF16)
    kc, vc = _pool(2, 1, 8, 16, BF16), _pool(2, 1, 8, 16, BF16)
    frequencies, zeros = gpuk.rope_frequencies(16, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    for slot, status in ((-1, cabi.OK), (16, cabi.ERR_INVALID_ARGUMENT), (1 << 40, cabi.ERR_INVALID_ARGUMENT), (-(1 << 63), cabi.OK)):
        q = gpuk.rope_paged(x[:, :1], x[:, 1:2], x[:, 2:], zeros, torch.tensor([3, slot, 5, slot], device="cuda"), frequencies, kc, vc)
        assert cabi.lib.gpuk_fp8_linear_status() == status
        assert q.isnan().all(-1).all(-1).tolist() == [False, True, False, True]
        assert [i for i in range(16) if vc.view(16, 16)[i].any()] == [3, 5] == [i for i in range(16) if kc.view(16, 16)[i].any()]


# ---- attention -------------------------------------------------------------------------------------------
class _Batch:
    """A ragged batch over pages in random order, its unused rows and pages full of `junk`."""

    def __init__(self, ctx, new, heads, kv, hd, page, dtype=BF16, seed=0, junk=float("nan"), order="hnd", spare=3, width=1, words=None, spread=1.5):
        rng, g = random.Random(seed), torch.Generator().manual_seed(seed)
        self.ctx, self.new, self.page, self.heads, self.kv, self.hd, self.dtype = ctx, new, page, heads, kv, hd, dtype
        need = [-(-(c + n) // page) for c, n in zip(ctx, new)]
        pages = sum(need) + spare
        ids = list(range(pages))
        rng.shuffle(ids)
        tables, at = [], 0
        for n in need:
            tables.append(ids[at:at + n] + [rng.choice([-1, 10 ** 9, ids[-1]]) for _ in range(max(need) + width - n)])
            at += n
        self.tables = _ints(tables)
        self.k, self.v = _pool(pages, kv, page, hd, dtype, order, junk), _pool(pages, kv, page, hd, dtype, order, junk)
        self.keys, self.values = [], []
        for i, (c, n) in enumerate(zip(ctx, new)):
            kk, vv = (torch.randn(c + n, kv, hd, generator=g).to(dtype).cuda() for _ in range(2))
            place = torch.arange(c + n, device="cuda")
            block = self.tables[i].long()[place // page]
            self.k[block, :, place % page], self.v[block, :, place % page] = kk, vv
            self.keys.append(kk.double()), self.values.append(vv.double())
        self.starts = _ints([sum(new[:i]) for i in range(len(new) + 1)])
        self.lens = _ints(ctx)
        self.q = (torch.randn(sum(new), heads, hd, generator=g) * spread).to(dtype).cuda()
        self.masks = None
        if words is not None:
            bits = [[rng.getrandbits(32 * words) & rng.getrandbits(32 * words) | (1 << j if rng.random() < 0.8 else 0) for j in range(n)] for n in new]
            self.bits = bits
            self.masks = _ints([[((b >> 32 * w & 0xffffffff) ^ 0x80000000) - 0x80000000 for w in range(words)] for row in bits for b in row]).view(-1, words)

    def seen(self, i):
        c, n = self.ctx[i], self.new[i]
        if self.masks is None:
            return torch.ones(n, c + n, dtype=torch.bool).tril(c).cuda()
        s = torch.ones(n, c + n, dtype=torch.bool)
        s[:, c:] = torch.tensor([[b >> j & 1 for j in range(n)] for b in self.bits[i]], dtype=torch.bool).view(n, n)
        return s.cuda()

    def run(self, **more):
        out = gpuk.paged_attention(self.q, self.k, self.v, self.tables, self.lens, self.starts, masks=self.masks, **more)
        _status_ok()
        return out

    def exact(self, scale=None):
        """Output and, for the bound, sum of weights times magnitudes and the weights' largest part."""
        scale = 1 / math.sqrt(self.hd) if scale is None else scale
        out, size = torch.zeros(self.q.shape, dtype=torch.float64, device="cuda"), torch.zeros(self.q.shape, dtype=torch.float64, device="cuda")
        group, at = self.heads // self.kv, 0
        for i, n in enumerate(self.new):
            seen = self.seen(i)
            for h in range(self.heads):
                k, v = self.keys[i][:, h // group], self.values[i][:, h // group]
                s = (self.q[at:at + n, h].double() @ k.T * scale).masked_fill(~seen, -math.inf)
                p = torch.softmax(s, -1).masked_fill(~seen, 0.0)
                dead = ~seen.any(-1)
                p[dead] = 0
                clean = torch.where(torch.isfinite(v), v, 0.0)
                o = p @ clean
                for j in torch.nonzero(~torch.isfinite(v).all(-1)).flatten().tolist():
                    o[seen[:, j]] += torch.where(torch.isfinite(v[j]), 0.0, v[j])
                out[at:at + n, h], size[at:at + n, h] = o, p @ clean.abs()
            at += n
        return out, size

    def check(self, got, scale=None):
        """Each weight is rounded once (half a step of it), and its fp32 value carries the error of a score of some tens, 2^-24 of it for each of the sums' roundings:
        2^-16 in all; the result is rounded once."""
        want, size = self.exact(scale)
        h = HALF_STEP[self.dtype]
        finite = torch.isfinite(want)
        bound = size * (h + 2.0 ** -15) + (want.abs() * h).nan_to_num(0, 0, 0) + 2.0 ** -24
        assert torch.equal(torch.isfinite(got), finite) and torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.double()[~finite & ~want.isnan()], want[~finite & ~want.isnan()])
        assert bool(((got.double() - want).abs() <= bound)[finite].all())


SHAPES = [(8, 1, 128, 16, BF16), (64, 8, 128, 64, BF16), (5, 5, 64, 8, F16), (28, 4, 128, 32, F16), (24, 8, 64, 128, BF16), (128, 1, 64, 256, BF16), (100, 1, 128, 16, F16)]


@pytest.mark.parametrize("heads,kv,hd,page,dtype", SHAPES)
@pytest.mark.parametrize("ctx,new", [([0], [1]), ([63, 64, 0], [1, 1, 1]), ([5, 127, 300, 0], [3, 1, 17, 64]), ([0, 130], [200, 33]), ([700, 12, 2000], [1, 0, 1]), ([3000], [5])])
def test_attention(ctx, new, heads, kv, hd, page, dtype):
    """Single tokens, runs that cross blocks and pages, requests with nothing new; tiles of one to 128 heads a token; keys in one part and in several."""
    b = _Batch(ctx, new, heads, kv, hd, page, dtype, seed=sum(ctx) + heads)
    got = b.run()
    b.check(got)
    assert torch.equal(got, b.run())
    if max(c + n for c, n in zip(ctx, new)) <= 256:      # in one part by the hint
        assert torch.equal(got, b.run(max_len=max(c + n for c, n in zip(ctx, new))))


@pytest.mark.parametrize("heads,kv,hd,page,dtype", SHAPES)
@pytest.mark.parametrize("ctx,new,words", [([0, 0], [1, 7], 1), ([60, 64, 1], [8, 33, 64], 2), ([1000, 3, 190], [13, 1, 130], 5), ([0, 65], [256, 2], 8), ([40], [70], 1)])
def test_attention_under_masks(ctx, new, words, heads, kv, hd, page, dtype):
    """Random bits: rows that see nothing at all, tokens beyond the masks, new keys that start anywhere in a block."""
    if words == 1 and new == [70]:
        b = _Batch(ctx, new, heads, kv, hd, page, dtype, seed=7, words=1)
        b.bits[0] = [x & 0xffffffff for x in b.bits[0]]
    else:
        b = _Batch(ctx, new, heads, kv, hd, page, dtype, seed=sum(new) + heads, words=words)
    b.check(b.run())


@pytest.mark.parametrize("heads,kv,hd,page,dtype", SHAPES[:5])
@pytest.mark.parametrize("ctx,new", [([300, 20, 1000, 5], [3, 0, 1, 0]), ([0] * 40, [1] * 40), ([5000, 0, 129], [1, 1, 1]), ([31], [1]), ([15, 16, 17, 2049], [0, 2, 0, 2])])
def test_attention_of_single_tokens(ctx, new, heads, kv, hd, page, dtype):
    """As many requests as tokens, or more: the kernel for single tokens, and what it does where a request has several or none."""
    b = _Batch(ctx, new, heads, kv, hd, page, dtype, seed=sum(ctx) + heads)
    got = b.run()
    b.check(got)
    assert torch.equal(got, b.run())
    for i, (c, n) in enumerate(zip(ctx, new)):      # a value of the last key that is not finite, and a key that is NaN
        if n:
            j = c + n - 1
            b.values[i][j, 0, 3] = math.inf
            b.v[int(b.tables[i, j // page]), 0, j % page, 3] = math.inf
    b.check(b.run())


@pytest.mark.parametrize("ctx,new", [([70, 500, 3], [2, 40, 9]), ([70, 500, 3] * 17, [1] * 51)])
@pytest.mark.parametrize("order", ["nhd", "wide"])
def test_attention_strides(order, ctx, new):
    b = _Batch(ctx, new, 16, 4, 128, 16, order=order)
    got = b.run()
    b.check(got)
    wide = torch.zeros(51, 24, 128, dtype=BF16, device="cuda")
    wide[:, 4:20] = b.q
    out = torch.full((51, 32, 128), 5.0, dtype=BF16, device="cuda")
    again = gpuk.paged_attention(wide[:, 4:20], b.k, b.v, b.tables, b.lens, b.starts, out=out[:, 8:24])
    assert torch.equal(again, got) and bool((out[:, :8] == 5).all()) and bool((out[:, 24:] == 5).all())
    tables = torch.full((len(ctx), 99), -7, dtype=torch.int32, device="cuda")
    tables[:, :b.tables.shape[1]] = b.tables
    assert torch.equal(gpuk.paged_attention(b.q, b.k, b.v, tables[:, :b.tables.shape[1]], b.lens, b.starts), got)


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("hd,dtype", [(128, BF16), (64, F16)])
def test_what_is_not_seen_does_not_reach_a_row(hd, dtype, masked):
    """Infinities and NaN among the new tokens' values and keys: rows that see them have them where the formula has, the others do not."""
    b = _Batch([61, 200, 0], [40, 9, 66], 8, 2, hd, 16, dtype, seed=3, words=3 if masked else None)
    for i, j, d, x in ((0, 61 + 7, 3, math.inf), (0, 61 + 20, 5, math.nan), (1, 203, 0, -math.inf), (2, 30, hd - 1, math.nan), (2, 65, 7, math.inf), (2, 31, hd - 1, -math.inf)):
        b.values[i][j, 1, d] = x
        b.v[int(b.tables[i, j // 16]), 1, j % 16, d] = x
    b.check(b.run())
    # a key that is NaN spoils exactly the rows that see it, of its kv head
    i, j = 2, 40
    b.k[int(b.tables[i, j // 16]), 0, j % 16] = math.nan
    got = b.run()
    rows = b.seen(i)[:, j]
    first = int(b.starts[i])
    assert bool(got[first:][rows][:, :4].isnan().all()) and not bool(got[first:][~rows][:, :4].isnan().any())


def test_scores_of_minus_infinity():
    """They weigh nothing beside others; a row that has only such is NaN, as a softmax has it; a row that sees no key is zeros."""
    b = _Batch([3], [3], 2, 1, 64, 16, words=1, seed=1)
    b.masks.copy_(_ints([[0], [2], [7]]))
    b.lens.zero_()
    b.q.fill_(1.0)
    b.k.fill_(-math.inf)
    b.k[int(b.tables[0, 0]), 0, 2] = 0.5
    got = b.run()
    assert not got[0].any() and bool(got[1].isnan().all())
    assert torch.equal(got[2], b.v[int(b.tables[0, 0]), 0, 2].expand(2, 64))


def test_large_scores_and_other_scales():
    for spread, scale in ((30.0, None), (1.0, 3.0), (1.0, 1e-4)):
        b = _Batch([400, 20], [5, 30], 8, 2, 128, 32, seed=5, spread=spread)
        want, size = b.exact(scale)
        got = b.run(scale=scale).double()
        # a score of s carries an error of s * 2^-22: sums of 128 exact products in fp32 (2^-24 each way) and the scaling
        most = float(b.q.float().abs().amax()) * 5 * 128 ** 0.5 * 3 * (scale or 0.09)
        assert bool(((got - want).abs() <= size * (2.0 ** -8 + max(1, most) * 2.0 ** -20) + want.abs() * 2.0 ** -8 + 1e-6).all())


def test_rows_behind_the_last_request_are_left():
    b = _Batch([100, 5], [1, 40], 8, 1, 128, 16)
    want = b.run()
    q = torch.cat([b.q, torch.full((13, 8, 128), math.nan, dtype=BF16, device="cuda")])
    out = torch.full_like(q, 3.0)
    gpuk.paged_attention(q, b.k, b.v, b.tables, b.lens, b.starts, out=out)
    _status_ok()
    assert torch.equal(out[:41], want) and bool((out[41:] == 3).all())


def test_the_bound_on_lengths_is_a_hint():
    """A smaller one than the lengths, and none: the keys are cut or not, the result is the formula's."""
    b = _Batch([5000, 1, 700], [3, 200, 9], 16, 2, 128, 32, seed=6)
    for bound in (None, 0, 1, 319, 320, 10 ** 12):
        b.check(b.run(max_len=bound))


@pytest.mark.parametrize("heads,kv,hd,page,dtype", SHAPES)
def test_the_bound_on_new_tokens_is_a_hint(heads, kv, hd, page, dtype):
    """Either kernel, with few and many requests, where the bound is true, too large or too small."""
    for ctx, new in [([500] + [0] * 30, [20] + [0] * 30), ([70, 3, 900, 0], [1, 1, 1, 1]), ([64, 300], [5, 130])]:
        b = _Batch(ctx, new, heads, kv, hd, page, dtype)
        for bound in (1, 2, max(new), 1 << 20):
            b.check(b.run(max_new=bound))
        # rows behind the last request, more of them than requests
        padded = torch.cat([b.q, b.q[:1].expand(len(new) + 3, -1, -1)])
        out = torch.full_like(padded, 3.0)
        gpuk.paged_attention(padded, b.k, b.v, b.tables, b.lens, b.starts, max_new=1, out=out)
        b.check(out[:sum(new)])
        assert bool((out[sum(new):] == 3).all())
    with pytest.raises(ValueError, match="new tokens"):
        b.run(max_new=0)


def test_more_tokens_than_the_table_holds():
    """Those behind the row's end have no keys: they see what there is; nothing is read outside the row."""
    b = _Batch([16], [40], 4, 2, 64, 16, spare=9)
    want = gpuk.paged_attention(b.q, b.k, b.v, b.tables[:, :2], b.lens, b.starts)
    _status_ok()
    full, b.keys, b.values = b.seen, [k[:32] for k in b.keys], [v[:32] for v in b.values]
    b.seen = lambda i: full(i)[:, :32]
    b.check(want)
    b.seen = lambda i: torch.ones(40, 32, dtype=torch.bool, device="cuda")
    b.check(gpuk.paged_attention(b.q, b.k, b.v, b.tables[:, :2], _ints([2 ** 31 - 1]), b.starts))


def test_many_requests_and_one_long_context():
    """Uneven work: one context is cut into many parts, the others into one; more requests than a warp has lanes."""
    rng = random.Random(2)
    ctx = [rng.randint(0, 90) for _ in range(69)] + [9000]
    b = _Batch(ctx, [rng.randint(0, 2) for _ in ctx[:-1]] + [1], 8, 2, 64, 16, F16, seed=4)
    b.check(b.run())


def test_a_cache_beyond_32_bits():
    """Elements of the pool that only 64-bit offsets reach."""
    pages, kv, page, hd = 70000, 8, 64, 64      # 2.3e9 values, 4.6 GB each
    k, v = (torch.zeros(pages, kv, page, hd, dtype=F16, device="cuda") for _ in range(2))
    far = [pages - 1, pages - 7]
    x = torch.randn(3, 100, kv, hd, generator=torch.Generator().manual_seed(0)).to(F16).cuda()
    slots = torch.tensor([far[i // page] * page + i % page for i in range(100)], device="cuda")
    zero = gpuk.rope_frequencies(64, device="cuda")
    positions = torch.zeros(100, dtype=torch.int64, device="cuda")
    q = gpuk.rope_paged(x[0], x[1], x[2], positions, slots, zero, k, v)
    tables, lens, starts = _ints([far + [-1]]), _ints([0]), _ints([0, 100])
    got = gpuk.paged_attention(q, k, v, tables, lens, starts)
    near = [c[far].clone() for c in (k, v)]
    assert torch.equal(got, gpuk.paged_attention(q, *near, _ints([[0, 1, -1]]), lens, starts)) and bool(got.any())
    assert torch.equal(near[0].transpose(1, 2).reshape(-1, kv, hd)[:100], x[1])
    out = gpuk.paged_keep(k, v, tables, _ints([10]), _ints([[3, 60]]))
    assert out.tolist() == [12] and torch.equal(v[far[0], :, 11], x[2][70]) and torch.equal(v[far[0], :, 10], x[2][13])
    _status_ok()


# ---- accepted paths --------------------------------------------------------------------------------------
@pytest.mark.parametrize("layers,kv,hd,page,dtype,order", [(None, 1, 64, 16, BF16, "hnd"), (3, 8, 128, 8, F16, "hnd"), (2, 5, 24, 1, BF16, "hnd"), (None, 3, 128, 64, BF16, "nhd")])
def test_keep(layers, kv, hd, page, dtype, order):
    """Paths of every length, rows that are moved onto what a later move reads, none, paths that stop ascending; all else keeps its bits."""
    g = torch.Generator().manual_seed(kv)
    pages, width = 60, -(-120 // page)
    lens = [0, 37, 50, 9, 63]
    tables = torch.full((5, width), -1, dtype=torch.int32)
    need = -(-(max(lens) + 40) // page)
    pages = 5 * need + 2
    tables[:, :need] = torch.randperm(pages, generator=g)[:5 * need].view(5, need)
    tables = tables.cuda()
    shape = (layers or 1, pages, kv, page, hd)
    k, v = (torch.randn(shape if order == "hnd" else (layers or 1, pages, page, kv, hd), generator=g).to(dtype).cuda() for _ in range(2))
    if order == "nhd":
        k, v = k.transpose(2, 3), v.transpose(2, 3)
    paths = [[0, 1, 2, 5, 6, 9, 10, 11, 12, 13, 20, 21, 22, 23, 24, 25, 26, 39], [2, 3, 4] + [-1] * 15, [-1] * 18, [0, 5, 5, 7] + [9] * 14, [7, 3] + [0] * 16]
    want = [k.clone(), v.clone()]
    after = []
    for i, path in enumerate(paths):
        n = 0
        while n < len(path) and path[n] > (path[n - 1] if n else -1):
            n += 1
        for j in range(n):
            a, b = lens[i] + path[j], lens[i] + j
            for c, src in zip(want, (k, v)):
                c[:, int(tables[i, b // page]), :, b % page] = src[:, int(tables[i, a // page]), :, a % page]
        after.append(lens[i] + n)
    got = gpuk.paged_keep(k if layers else k[0], v if layers else v[0], tables, _ints(lens), _ints(paths))
    assert got.tolist() == after and torch.equal(k, want[0]) and torch.equal(v, want[1])


def test_keep_at_the_table_s_end():
    """Nodes behind the row's last page, and pages that are none, move nothing."""
    k = torch.randn(2, 1, 8, 16).to(BF16).cuda()
    v, want = k.clone(), k.clone()
    want[1, :, 2] = k[1, :, 3]
    got = gpuk.paged_keep(k, v, _ints([[1, -1], [0, 5]]), _ints([2, 7]), _ints([[1, 9, 400], [1, 2, 3]]))
    assert got.tolist() == [5, 10] and torch.equal(k, want) and torch.equal(v, want)


# ---- views of one allocation -----------------------------------------------------------------------------
@pytest.mark.parametrize("order", ["pages", "rows", "layers"])
def test_keys_and_values_of_one_allocation(order):
    """Keys and values as the two halves of each page, of each row, or of the whole pool: the same bits as in pools of their own."""
    pages, kv, page, hd, n = 9, 2, 16, 64, 40
    both = torch.zeros({"pages": (pages, 2, kv, page, hd), "rows": (pages, kv, page, 2, hd), "layers": (2, pages, kv, page, hd)}[order], dtype=BF16, device="cuda")
    k, v = both.unbind({"pages": 1, "rows": 3, "layers": 0}[order])
    own_k, own_v = torch.zeros_like(k, memory_format=torch.contiguous_format), torch.zeros_like(k, memory_format=torch.contiguous_format)
    g = torch.Generator().manual_seed(5)
    x, q = torch.randn(2, n, kv, hd, generator=g).to(BF16).cuda(), torch.randn(n, 6, hd, generator=g).to(BF16).cuda()
    tables, lens, f = _ints([[7, 2, 4, -1]]), _ints([0]), gpuk.rope_frequencies(hd, device="cuda")
    at = torch.arange(n, device="cuda")
    slots = tables[0].long()[at // page] * page + at % page
    got = []
    for kc, vc in ((k, v), (own_k, own_v)):
        rotated = gpuk.rope_paged(q, x[0], x[1], at, slots, f, kc, vc)
        out = [rotated] + [gpuk.paged_attention(rotated[a:], kc, vc, tables, _ints([a]), _ints([0, n - a])) for a in (0, n - 1)]
        got.append(out + [gpuk.paged_keep(kc, vc, tables, lens, _ints([[1, 5, 30]])), kc.clone(), vc.clone()])
    _status_ok()
    assert all(torch.equal(a, b) for a, b in zip(*got)) and bool(got[0][-1].any())


def test_queries_in_place_beside_their_keys():
    """Queries of a joint projection are rotated where they are; what would be read behind a write, or written twice, is refused."""
    x = torch.randn(5, 12, 64, generator=torch.Generator().manual_seed(2)).to(BF16).cuda()
    at, f = torch.arange(5, device="cuda"), gpuk.rope_frequencies(64, device="cuda")
    k, v = _pool(1, 4, 8, 64, BF16), _pool(1, 4, 8, 64, BF16)
    parts = [x.split([4, 4, 4], dim=1), x.view(5, 4, 3, 64).unbind(2)]      # heads one after another, and each with its key and value
    for i in range(2):
        want = gpuk.rope_paged(*parts[i], at, at, f, k, v)
        held, before = (k.clone(), v.clone()), x.clone()
        q = parts[i][0]
        assert torch.equal(gpuk.rope_paged(*parts[i], at, at, f, k, v, out=q), want) and torch.equal(q, want)
        assert torch.equal(k, held[0]) and torch.equal(v, held[1])
        q.copy_((before.split([4, 4, 4], dim=1)[0] if i == 0 else before.view(5, 4, 3, 64)[:, :, 0]))
        assert torch.equal(x, before)
    q, kx, vx = parts[0]
    twice = torch.zeros(400, dtype=BF16, device="cuda").as_strided((5, 4, 64), (64, 8, 1))
    for call, text in [(lambda: gpuk.rope_paged(q, q, vx, at, at, f, k, v, out=q), "overlaps k or v"), (lambda: gpuk.rope_paged(q, x[:, 3:7], vx, at, at, f, k, v, out=q), "overlaps k or v"),
                       (lambda: gpuk.rope_paged(q, kx, vx, at, at, f, k, k), "overlap"), (lambda: gpuk.rope_paged(q, kx, vx, at, at, f, k[:, :, :1].expand(1, 4, 8, 64), v[:, :, :1].expand(1, 4, 8, 64)), "repeat"),
                       (lambda: gpuk.rope(q, at, f, out=twice), "repeats"), (lambda: gpuk.rope(q, at, f, out=twice[:1].expand(5, 4, 64)), "repeats")]:
        with pytest.raises(RuntimeError, match=text):
            call()
    torch.cuda.synchronize()
