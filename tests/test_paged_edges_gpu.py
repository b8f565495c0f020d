"""The paged cache at its edges: rows of the table that end inside a tile, pools that run out, tokens without a place, and callers that want to see what is computed."""
import random

import pytest
import torch

import gpuk_b200 as gpuk
from tests.test_paged_gpu import BF16, F16, _Batch, _ints, _status_ok

pytestmark = pytest.mark.gpu


# ---- tables that end inside a tile ---------------------------------------------------------------------------
def _cut(ctx, new, heads, kv, hd, page, width, dtype=BF16, **more):
    """A batch whose table has fewer pages than some requests' tokens: what a token sees ends with the row."""
    b = _Batch(ctx, new, heads, kv, hd, page, dtype, **more)
    room, full = width * page, b.seen
    b.tables = b.tables[:, :width]
    b.keys, b.values = [k[:room] for k in b.keys], [v[:room] for v in b.values]
    b.seen = lambda i: full(i)[:, :room]
    return b


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("heads,kv,hd,page,width,ctx,new,dtype", [(8, 1, 128, 16, 2, [16], [64], BF16), (64, 8, 128, 16, 5, [0, 3], [200, 2], BF16), (8, 1, 64, 8, 1, [0], [40], F16),
                                                                 (64, 8, 64, 32, 3, [90, 96, 7], [150, 33, 60], F16), (128, 1, 128, 8, 9, [70], [9], BF16), (5, 5, 64, 8, 17, [0], [250], BF16),
                                                                 (16, 2, 128, 64, 1, [0, 64], [70, 20], BF16)])
def test_tiles_behind_the_table_s_end(heads, kv, hd, page, width, ctx, new, dtype, masked):
    """Tiles that begin behind the last key of the row: keys that are not there weigh nothing, whichever kernel takes the call."""
    b = _cut(ctx, new, heads, kv, hd, page, width, dtype, seed=heads + page, words=8 if masked else None)
    got = b.run()
    b.check(got)
    if not masked:
        b.check(b.run(max_new=1))


# ---- pools that run out ------------------------------------------------------------------------------------
def _state(cache):
    """The pages of every request and of the list, each once."""
    held = [[int(x) for x in row[:n]] for row, n in zip(cache.tables.tolist(), cache.held.tolist())]
    free = cache.free[:int(cache.free_count[0])].tolist()
    return held, free


def _write(cache, plan, g, heads=2):
    """Random keys and values of the new tokens into their slots; returns them."""
    n, kv, hd = plan.slots.shape[0], cache.k.shape[2], cache.k.shape[4]
    x = torch.randn(3, n, max(heads, kv), hd, generator=g).to(cache.k.dtype).cuda()
    zero = torch.zeros(n, dtype=torch.int64, device="cuda")      # no rotation
    q = gpuk.rope_paged(x[0, :, :heads].contiguous(), x[1, :, :kv], x[2, :, :kv], zero, plan.slots, gpuk.rope_frequencies(hd, device="cuda"), cache.k[0], cache.v[0])
    return x[0, :, :heads], q, x[1, :, :kv], x[2, :, :kv]


def _attended(q, keys, values):
    """One token over the keys given, in 64 bits."""
    s = torch.einsum("hd,nhd->hn", q.double(), keys.double()) / q.shape[-1] ** 0.5
    return torch.einsum("hn,nhd->hd", torch.softmax(s, -1), values.double())


@pytest.mark.parametrize("step", ["append", "keep"])
def test_tokens_without_a_page_do_not_become_cached(step):
    """The pool runs out in the middle of a request's new tokens.  What has no page is not counted as cached, so that a page that comes free later, with keys of its last owner, is not taken for
    it; the next token goes where the cached ones end and sees them and itself."""
    g = torch.Generator().manual_seed(3)
    cache = gpuk.PagedKVCache(1, 4, 8, 2, 64, 2, 6)
    first = _ints([10, 7])
    plan = cache.plan(first, 17)
    _, _, k0, v0 = _write(cache, plan, g)
    cache.append(first)
    assert cache.lens.tolist() == [10, 7] and cache.held.tolist() == [2, 1]
    # 14 more tokens of the first request: 6 and 8 of them have pages; a chain, so that both steps keep them all
    more = _ints([20, 0])
    plan = cache.plan(more, 20, parents=_ints(list(range(-1, 19))), max_new=20)
    assert plan.free_count.tolist() == [0, 1] and plan.slots[14:].tolist() == [-1] * 6
    _, q, k1, v1 = _write(cache, plan, g)
    assert bool(q[14:].isnan().all())
    if step == "append":
        cache.append(more)
    else:
        cache.keep(_ints([list(range(20)), [-1] * 20]))
    assert cache.lens.tolist() == [24, 7]
    # the second request ends and its page, full of its keys, goes to the first
    cache.release([1])
    one = _ints([1, 0])
    plan = cache.plan(one, 1)
    assert plan.free_count.tolist() == [0, 0] and plan.positions.tolist() == [24] and cache.held.tolist() == [4, 0]
    raw, q, k2, v2 = _write(cache, plan, g)
    got = gpuk.paged_attention(q, cache.k[0], cache.v[0], cache.tables, cache.lens, plan.starts)
    want = _attended(q[0], torch.cat([k0[:10], k1[:14], k2]), torch.cat([v0[:10], v1[:14], v2]))
    # weights and the result rounded to bf16 once each, sums of magnitudes of a few units
    assert float((got[0].double() - want).abs().amax()) <= 2.0 ** -7 * 4
    cache.append(one)
    assert cache.lens.tolist() == [25, 0]
    _status_ok()


def test_a_path_ends_at_its_first_token_without_a_page():
    """Accepted nodes in front of it are kept, those behind it are not, even where the rows that they would move to have pages; a request with all of its pages keeps its path."""
    g = torch.Generator().manual_seed(4)
    cache = gpuk.PagedKVCache(1, 5, 8, 2, 64, 2, 6)
    plan = cache.plan(_ints([4, 9]), 13)
    _write(cache, plan, g)
    cache.append(_ints([4, 9]))
    assert cache.held.tolist() == [1, 2]
    # trees of 26 and 5 nodes behind 4 and 9 tokens: 30 tokens want four pages, of which three are to be had
    plan = cache.plan(_ints([26, 5]), 31, parents=_ints([-1] + [0] * 25 + [-1, 0, 0, 1, 3]), max_new=26)
    assert cache.held.tolist() == [3, 2] and plan.free_count.tolist() == [0, 1] and plan.slots[:26].tolist().index(-1) == 20
    _, _, k, v = _write(cache, plan, g)
    cache.keep(_ints([[0, 3, 21, 23], [0, 1, 3, 4]]))
    assert cache.lens.tolist() == [6, 13]
    for i, (c, at) in enumerate(((4, [0, 3]), (9, [26, 27, 29, 30]))):
        for j, node in enumerate(at):
            page = int(cache.tables[i, (c + j) // 8])
            assert torch.equal(cache.k[0, page, :, (c + j) % 8], k[node]) and torch.equal(cache.v[0, page, :, (c + j) % 8], v[node])


@pytest.mark.parametrize("seed", range(4))
def test_a_pool_that_is_always_short(seed):
    """Random steps of requests that want more than there is: lengths never pass the pages that are held, no page is lost or twice, and every cached row holds what was written for it."""
    rng, g = random.Random(seed), torch.Generator().manual_seed(seed)
    cache = gpuk.PagedKVCache(1, 12, 8, 1, 64, 4, 5)
    texts = [[] for _ in range(4)]      # the values of the cached tokens
    for _ in range(25):
        new = [rng.choice([0, 1, 1, 5, 12]) for _ in range(4)]
        for i in range(4):
            if rng.random() < 0.15:
                cache.release([i])
                texts[i] = []
        total = sum(new)
        tree = rng.random() < 0.5
        plan = cache.plan(_ints(new), total, parents=_ints([p for n in new for p in range(-1, n - 1)]) if tree else None, max_new=12 if tree else 0)
        slots, starts = plan.slots.tolist(), plan.starts.tolist()
        if total:
            _, _, _, v = _write(cache, plan, g)
        there = [[j for j in range(n) if slots[starts[i] + j] >= 0] for i, n in enumerate(new)]
        if tree:      # every other node of the chain: any ascending list is a path to the call
            paths = [list(range(rng.randint(0, 1), n, rng.randint(1, 2))) for n in new]
            cache.keep(_ints([p + [-1] * (12 - len(p)) for p in paths]))
            kept = [[j for j in p if j in there[i]] for i, p in enumerate(paths)]
        else:
            cache.append(_ints(new))
            kept = there
        for i in range(4):
            texts[i] += [v[starts[i] + j, 0] for j in kept[i]]
        assert cache.lens.tolist() == [len(t) for t in texts]
        held, free = _state(cache)
        assert sorted(sum(held, []) + free) == list(range(12)) and all(len(t) <= 8 * len(h) for t, h in zip(texts, held))
        for t, h in zip(texts, held):
            for j, row in enumerate(t):
                assert torch.equal(cache.v[0, h[j // 8], 0, j % 8], row)


def test_lengths_that_are_held_stay_as_they_are():
    """Fewer tokens appended than were planned, none, and none with negative counts, which a plan takes for none; a request that fills its pages to the end."""
    cache = gpuk.PagedKVCache(1, 9, 8, 1, 64, 3, 4)
    cache.plan(_ints([16, 3, -5]), 19)
    cache.append(_ints([16, 2, -5]))
    assert cache.lens.tolist() == [16, 2, 0]
    cache.plan(_ints([16, 5, 0]), 21)
    cache.append(_ints([16, 5, 0]))
    assert cache.lens.tolist() == [32, 7, 0] and cache.held.tolist() == [4, 1, 0]


# ---- callers that want to see what is computed ------------------------------------------------------------------
def _calls():
    """The five entry points on small arguments, each writing nothing that another reads."""
    b = _Batch([10], [2], 4, 2, 64, 16)
    ints = [_ints([3]), _ints([1]), _ints([[0, -1]]), _ints([1]), _ints([2, 3, 0, 0]), _ints([2, 0])]
    at, f = torch.arange(2, device="cuda"), gpuk.rope_frequencies(64, device="cuda")
    return b, {"paged_plan": lambda: gpuk.paged_plan(*ints, 16, 1), "rope": lambda: gpuk.rope(b.q, at, f),
               "rope_paged": lambda: gpuk.rope_paged(b.q, b.q[:, :2], b.q[:, 2:], at, at, f, b.k, b.v),
               "paged_attention": lambda: gpuk.paged_attention(b.q, b.k, b.v, b.tables, b.lens, b.starts),
               "paged_keep": lambda: gpuk.paged_keep(b.k, b.v, b.tables, b.lens, _ints([[0]]))}


@pytest.mark.parametrize("name", ["paged_plan", "rope", "rope_paged", "paged_attention", "paged_keep"])
def test_modes_and_tracers_are_refused(name):
    """A dispatch mode, a trace and a transform would not see the call: a trace would hold its result as a constant and never write the pages."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    b, calls = _calls()
    with pytest.raises(RuntimeError, match="mode"), Watch():
        calls[name]()
    with pytest.raises(RuntimeError, match="mode"):
        torch.jit.trace(lambda x: x + calls[name]()[0].float().sum(), (torch.zeros(1, device="cuda"),), check_trace=False)
    with pytest.raises(RuntimeError, match="mode"):
        torch.func.vmap(lambda x: calls[name]()[0] * x)(torch.ones(2, device="cuda"))
    # what only says where new tensors go sees nothing of a call and keeps none from it
    with torch.device("cuda"):
        calls[name]()
    with torch.inference_mode():
        calls[name]()
    with torch.autocast("cuda"):
        calls[name]()
    torch.cuda.synchronize()


@pytest.mark.parametrize("grad", [True, False])
def test_tangents_are_refused(grad):
    """A forward-mode tangent would be dropped; without forward mode there is none to drop."""
    import torch.autograd.forward_ad as fwd

    b, _ = _calls()
    at, f = torch.arange(2, device="cuda"), gpuk.rope_frequencies(64, device="cuda")
    with torch.set_grad_enabled(grad), fwd.dual_level():
        dual = fwd.make_dual(b.q, torch.ones_like(b.q))
        with pytest.raises(RuntimeError, match="tangent"):
            gpuk.paged_attention(dual, b.k, b.v, b.tables, b.lens, b.starts)
        with pytest.raises(RuntimeError, match="tangent"):
            gpuk.rope(dual, at, f)
        with pytest.raises(RuntimeError, match="tangent"):
            gpuk.rope_paged(dual, b.q[:, :2], b.q[:, 2:], at, at, f, b.k, b.v)
        gpuk.paged_attention(b.q, b.k, b.v, b.tables, b.lens, b.starts)      # tangents elsewhere are no matter
        with fwd._set_fwd_grad_enabled(False):
            gpuk.paged_attention(dual, b.k, b.v, b.tables, b.lens, b.starts)


# ---- tokens without a place ----------------------------------------------------------------------------------
@pytest.mark.parametrize("fp8", [False, True])
def test_logits_of_tokens_without_a_slot(fp8):
    """Trees larger than the table's row, without cached tokens, so that a node behind its end sees no key at all, and trees that found no page: NaN all the same; the others are numbers."""
    from tests.test_paged_decoder_gpu import _decoder

    own = not torch.distributed.is_initialized()
    if own:
        torch.distributed.init_process_group("gloo", store=torch.distributed.HashStore(), rank=0, world_size=1)
    try:
        model = _decoder(gpuk.GPUKDistEnv(group=None, device_id=0), fp8)
        for pages, requests, per, new in [(9, 2, 1, [20, 6]), (2, 3, 4, [20, 20, 3])]:
            cache = model.paged_cache(pages=pages, requests=requests, pages_per_request=per, page_size=16)
            plan = cache.plan(_ints(new), sum(new), parents=_ints([-1] * sum(new)), max_new=20)
            without = plan.slots < 0
            assert bool(without.any()) and not bool(without.all())
            logits = model.forward_paged(torch.arange(sum(new), device="cuda"), cache, plan)
            assert torch.equal(logits.isnan().all(-1), without) and torch.equal(logits.isnan().any(-1), without)
        _status_ok()
    finally:
        if own:
            torch.distributed.destroy_process_group()


# ---- clusters that have no place ------------------------------------------------------------------------------
@pytest.mark.parametrize("ctas", [1, 2, 4, 8, 16])
def test_plans_by_smaller_clusters(ctas):
    """A part of a GPU may have no place for sixteen CTAs that meet: a plan by any number of them is the same."""
    from gpuk_b200 import cabi
    from tests.test_paged_gpu import _check_plan, _random_state

    cabi.check(cabi.lib.gpuk_set_tuning(b"paged_plan_ctas", ctas))
    try:
        for batch, page, ctx, new, spare, slack in [(3, 16, 40, 20, 20, 5), (7, 16, 50, 9000, 5000, 3), (1030, 32, 300, 40, 3500, 0)]:
            _check_plan(*_random_state(random.Random(batch), batch, page, ctx, new, spare, slack))
        rng = random.Random(ctas)
        for batch, new in ((300, 64), (90, 256)):
            state = _random_state(rng, batch, 16, 100, new, batch * new // 10, 2)
            parents = [rng.choice([-1, j - 1, rng.randint(-1, max(j - 1, -1))]) for n in state[1] for j in range(n)]
            _check_plan(*state, parents=parents + [-1, -1], max_new=new)
    finally:
        cabi.check(cabi.lib.gpuk_set_tuning(b"paged_plan_ctas", 0))


# ---- rounded weights -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("hd,dtype", [(128, BF16), (64, BF16), (128, F16), (64, F16)])
def test_a_weight_that_dominates_moves_nothing_by_its_rounding(hd, dtype):
    """Two keys of different blocks carry each row, the second with a weight of up to 2^7 that the operands' type does not hold, and all values are alike: what comes out is that value, as
    the sum holds the weight as it was multiplied.  Other keys weigh 2^-32 or less each beside the first; sums of two products and the quotient are off by some 2^-22, which no value's rounding sees."""
    heads, ctx = 96, 190
    b = _Batch([ctx], [2], heads, 1, hd, 64, dtype)
    g = torch.Generator().manual_seed(hd)
    value = torch.randn(hd, generator=g).to(dtype).cuda()
    b.v[:] = value
    b.k[:] = 0
    b.k[..., 0] = -64.0
    b.k[int(b.tables[0, 0]), 0, 5] = 0
    b.k[int(b.tables[0, 2]), 0, 2, 0] = 1.0
    b.q[:] = 0
    # log2 of the second weight: 0.5 to 6.9, so the others are at -32 and below, beside the two
    b.q[..., 0] = (torch.rand(2, heads, generator=g) * 6.4 + 0.5).cuda().to(dtype)
    got = b.run(scale=0.6931471805599453)
    assert torch.equal(got, value.expand(2, heads, hd))


# ---- many requests, and none ---------------------------------------------------------------------------------
@pytest.mark.parametrize("batch,most", [(1000, 1), (4096, 1), (1500, 3)])
def test_attention_of_thousands_of_requests(batch, most):
    """Each lane of the border search looks after a hundred of them; single tokens, and a few each, against a padded batch in 64 bits."""
    rng, g = random.Random(batch), torch.Generator(device="cuda").manual_seed(batch)
    page, kv, heads, hd, longest = 16, 2, 4, 64, 40
    ctx, new = [rng.randint(0, longest - most) for _ in range(batch)], [rng.randint(0, most) if rng.random() < 0.5 else most for _ in range(batch)]
    ctx[7], width = 700, 48      # one of them is cut into parts
    total = sum(new)
    pages = sum(-(-(c + n) // page) for c, n in zip(ctx, new))
    order, tables, at = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).tolist(), [], 0
    for c, n in zip(ctx, new):
        need = -(-(c + n) // page)
        tables.append(order[at:at + need] + [-1] * (width - need))
        at += need
    k, v = (torch.randn(pages, kv, page, hd, generator=g, device="cuda").to(BF16) for _ in range(2))
    q = torch.randn(total, heads, hd, generator=g, device="cuda").to(BF16)
    starts = torch.tensor([0] + new).cumsum(0).int().cuda()
    t, lens = _ints(tables), _ints(ctx)
    got = gpuk.paged_attention(q, k, v, t, lens, starts)
    _status_ok()
    request = torch.repeat_interleave(torch.arange(batch, device="cuda"), torch.tensor(new, device="cuda"))
    index = torch.arange(total, device="cuda") - starts[request]
    for part in torch.arange(total, device="cuda").split(512):
        r = request[part]
        kk, vv = (c[t[r].long().clamp(min=0)].transpose(2, 3).reshape(len(r), width * page, kv, hd).repeat_interleave(heads // kv, 2).double() for c in (k, v))
        s = torch.einsum("thd,tnhd->thn", q[part].double(), kk) / hd ** 0.5
        seen = torch.arange(width * page, device="cuda") <= (lens[r] + index[part])[:, None]
        p = torch.softmax(s.masked_fill(~seen[:, None], float("-inf")), -1)
        want, size = torch.einsum("thn,tnhd->thd", p, vv), torch.einsum("thn,tnhd->thd", p, vv.abs())
        # each weight and the result are rounded once
        assert bool(((got[part].double() - want).abs() <= size * (2.0 ** -8 + 2.0 ** -15) + want.abs() * 2.0 ** -8 + 2.0 ** -24).all())


@pytest.mark.parametrize("fp8", [False, True])
def test_a_step_of_nothing(fp8):
    """A server whose requests have all ended: no rows, no logits, and nothing changes."""
    from tests.test_paged_decoder_gpu import _decoder

    own = not torch.distributed.is_initialized()
    if own:
        torch.distributed.init_process_group("gloo", store=torch.distributed.HashStore(), rank=0, world_size=1)
    try:
        model = _decoder(gpuk.GPUKDistEnv(group=None, device_id=0), fp8)
        cache = model.paged_cache(pages=4, requests=2, pages_per_request=2, page_size=16)
        none = _ints([0, 0])
        logits = model.forward_paged(torch.zeros(0, dtype=torch.int64, device="cuda"), cache, cache.plan(none, 0))
        cache.append(none)
        assert logits.shape == (0, 512) and cache.lens.tolist() == [0, 0] and cache.free_count.tolist() == [4, 0]
        _status_ok()
    finally:
        if own:
            torch.distributed.destroy_process_group()


def test_trees_without_nodes():
    """A plan for trees of which there are none, and what follows it: pages still come back."""
    cache = gpuk.PagedKVCache(1, 4, 8, 2, 64, 2, 3)
    cache.plan(_ints([9, 3]), 12)
    cache.append(_ints([9, 3]))
    cache.release([0])
    plan = cache.plan(_ints([0, 0]), 0, parents=_ints([]), max_new=5)
    assert plan.masks.shape == (0, 1) and plan.starts.tolist() == [0, 0, 0] and cache.held.tolist() == [0, 1] and cache.free_count.tolist() == [3, 0]
    q = torch.zeros(0, 4, 64, dtype=BF16, device="cuda")
    q = gpuk.rope_paged(q, q[:, :2], q[:, :2], plan.positions, plan.slots, gpuk.rope_frequencies(64, device="cuda"), cache.k[0], cache.v[0])
    assert gpuk.paged_attention(q, cache.k[0], cache.v[0], cache.tables, cache.lens, plan.starts, masks=plan.masks).shape == (0, 4, 64)
    cache.keep(_ints([[-1], [-1]]))
    assert cache.lens.tolist() == [0, 3]
    empty = gpuk.paged_plan(_ints([]), _ints([]), _ints([]).view(0, 4), _ints([]), _ints([3, 2]), _ints([2, 0]), 16, 2, parents=_ints([7, -1]), max_new=40)
    assert empty.slots.tolist() == [-1, -1] and not bool(empty.masks.any()) and empty.masks.shape == (2, 2)
