"""The paged cache in use: a decoder over requests of different lengths, trees of drafts verified and kept, the same from a captured graph; streams, and what the calls refuse."""
import random

import pytest
import torch
import torch.distributed as dist

import gpuk_b200 as gpuk
from gpuk_b200 import cabi
from gpuk_b200.tp_model import DecoderArgs, TPDecoder
from tests.test_paged_gpu import _Batch, _ints

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    own = not dist.is_initialized()
    if own:
        dist.init_process_group("gloo", store=dist.HashStore(), rank=0, world_size=1)
    yield gpuk.GPUKDistEnv(group=None, device_id=0)
    if own:
        dist.destroy_process_group()


def _decoder(env, fp8=False, **more):
    args = DecoderArgs(dim=1024, n_layers=2, n_heads=8, n_kv_heads=2, ffn_dim=2048, vocab_size=512, max_seq_len=512, **more)
    return TPDecoder(args, env, device="cuda:0", fp8=fp8, max_batch=1)


def _alone(model, tokens):
    """Logits of a sequence by itself, over the contiguous cache."""
    n = len(tokens)
    return model.forward(torch.tensor([tokens], device="cuda"), torch.arange(n, device="cuda"), cache_len=n)[0].float()


def _near(got, want, fp8=False):
    """Both run in bf16 and round at the same places, up to the order of the sums in attention and in the projections, which may turn a rounding (2^-8 of a value) at each of
    the some ten places of a layer: in the norm over many logits, far below 2^-8 times the square root of twenty such places, 1.8e-2; FP8 codes a step of 2^-3 apart in a few
    places come on top."""
    got, want = got.float(), want.float()
    assert torch.isfinite(got).all()
    assert float((got - want).norm()) <= (0.06 if fp8 else 0.02) * float(want.norm())


@pytest.mark.parametrize("fp8,more", [(False, {}), (True, {}), (False, {"rope_scaling": {"kind": "yarn", "factor": 8.0, "low": 1.0, "high": 32.0, "original": 64}})])
def test_a_server(env, fp8, more):
    """Prompts of any length at once, a decode step for all, trees of drafts, the accepted path kept, the next step on top of it; a request ends and another takes its pages."""
    model = _decoder(env, fp8, **more)
    rng = random.Random(5)
    text = [[rng.randrange(512) for _ in range(n)] for n in (1, 70, 33, 128)]
    cache = model.paged_cache(pages=30, requests=4, pages_per_request=12, page_size=16)

    def step(new, parents=None, max_new=0):
        lens = _ints([len(n) for n in new])
        flat = torch.tensor([t for n in new for t in n], device="cuda")
        plan = cache.plan(lens, len(flat), parents=None if parents is None else _ints([p for n in parents for p in n]), max_new=max_new)
        logits = model.forward_paged(flat, cache, plan)
        cabi.check(cabi.lib.gpuk_fp8_linear_status())
        assert cache.free_count[1] == 0
        return logits.split([len(n) for n in new]), lens

    got, lens = step(text)
    cache.append(lens)
    for g, t in zip(got, text):
        _near(g, _alone(model, t), fp8)
    more_tokens = [[rng.randrange(512)] for _ in text]
    got, lens = step(more_tokens)
    cache.append(lens)
    text = [t + m for t, m in zip(text, more_tokens)]
    for g, t in zip(got, text):
        _near(g, _alone(model, t)[-1:], fp8)
    # trees: each node's logits are those of its path by itself
    parents = [[-1, 0, 0, 1, 1, 2, 3], [-1], [-1, 0, 1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13, 14, 15, 16, 17, 18], [-1, 0, 0, 0, 3, 3, 2, 1, 7, 4]]
    drafts = [[rng.randrange(512) for _ in p] for p in parents]
    got, _ = step(drafts, parents, max_new=20)
    paths = [[0, 1, 4], [0], [0, 1, 2, 3, 4, 5, 6, 7, 8], [0, 3, 4, 9]]
    for g, t, d, p in zip(got, text, drafts, parents):
        for node in (len(p) - 1, len(p) // 2):
            path = [node]
            while p[path[0]] >= 0:
                path.insert(0, p[path[0]])
            _near(g[path], _alone(model, t + [d[j] for j in path])[-len(path):], fp8)
    cache.keep(_ints([p + [-1] * (9 - len(p)) for p in paths]))
    text = [t + [d[j] for j in p] for t, d, p in zip(text, drafts, paths)]
    assert cache.lens.tolist() == [len(t) for t in text]
    # the last ends; the first goes on with a long prompt that needs its pages
    cache.release([3])
    more_tokens = [[rng.randrange(512) for _ in range(150)], [7], [rng.randrange(512)], []]
    got, lens = step(more_tokens)
    cache.append(lens)
    text = [t + m for t, m in zip(text, more_tokens)]
    for g, t, m in zip(got[:3], text, more_tokens):
        _near(g, _alone(model, t)[-len(m):], fp8)
    assert cache.held.tolist() == [-(-len(t) // 16) for t in text[:3]] + [0]
    assert int(cache.free_count[0]) == 30 - int(cache.held.sum())
    everywhere = [int(x) for row, n in zip(cache.tables.tolist(), cache.held.tolist()) for x in row[:n]] + cache.free[:int(cache.free_count[0])].tolist()
    assert sorted(everywhere) == list(range(30))      # no page twice, none lost


def test_a_server_from_a_graph(env):
    """One decode step captured: lengths, tables and pages move on in place with each replay; two graphs of two caches run side by side."""
    model = _decoder(env)
    caches, graphs, tokens, logits, texts = [], [], [], [], []
    rng = random.Random(1)
    ones = _ints([1, 1, 1])
    for _ in range(2):
        cache = model.paged_cache(pages=40, requests=3, pages_per_request=10, page_size=16)
        text = [[rng.randrange(512) for _ in range(n)] for n in (300 // 3, 14, 31)]
        lens = _ints([len(t) for t in text])
        total = sum(map(len, text))
        plan = cache.plan(lens, total)
        model.forward_paged(torch.tensor([t for s in text for t in s], device="cuda"), cache, plan)
        cache.append(lens)
        inp = torch.zeros(4, dtype=torch.int64, device="cuda")      # a row more than there are requests

        def step(cache=cache, inp=inp):
            plan = cache.plan(ones, 4)
            out = model.forward_paged(inp, cache, plan)
            cache.append(ones)
            return out
        state = [t.clone() for t in (cache.lens, cache.held, cache.free_count, cache.tables, cache.free)]
        step()
        for t, s in zip((cache.lens, cache.held, cache.free_count, cache.tables, cache.free), state):
            t.copy_(s)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        caches.append(cache), graphs.append(graph), tokens.append(inp), logits.append(out), texts.append(text)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for i in range(20):      # over the border of a page for each request
        fresh = [[rng.randrange(512) for _ in range(3)] for _ in range(2)]
        for s, g, inp, f in zip(streams, graphs, tokens, fresh):
            inp[:3] = torch.tensor(f, device="cuda")
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for text, f in zip(texts, fresh):
            for t, x in zip(text, f):
                t.append(x)
        if i in (0, 18, 19):
            for text, out in zip(texts, logits):
                for t, row in zip(text, out):
                    _near(row[None], _alone(model, t)[-1:])
    cabi.check(cabi.lib.gpuk_fp8_linear_status())


def test_two_calls_at_once_and_another_stream():
    """Calls on two streams share nothing; one on a side stream is ordered as PyTorch orders it."""
    a, b = _Batch([3000, 20], [4, 70], 8, 1, 128, 16, seed=1), _Batch([2500], [3], 64, 8, 64, 32, torch.float16, seed=2)
    want = a.run(), b.run()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    outs = []
    for _ in range(10):
        for s, batch in zip(streams, (a, b)):
            with torch.cuda.stream(s):
                outs.append(gpuk.paged_attention(batch.q, batch.k, batch.v, batch.tables, batch.lens, batch.starts))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i % 2]) for i, o in enumerate(outs))


def test_capture_of_a_join():
    """A call with parts, captured: its workspace belongs to the graph; replayed with other lengths and queries."""
    b = _Batch([4000, 100], [2, 1], 16, 2, 128, 64, seed=3)
    b.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = gpuk.paged_attention(b.q, b.k, b.v, b.tables, b.lens, b.starts)
    for ctx in ([4000, 100], [11, 80], [2222, 0]):
        # the new tokens are those behind the shorter contexts
        b.ctx = ctx
        b.keys, b.values = [k for k in b.keys], [v for v in b.values]
        b.lens.copy_(_ints(ctx))
        b.q.normal_()
        graph.replay()
        torch.cuda.synchronize()
        eager = gpuk.paged_attention(b.q, b.k, b.v, b.tables, b.lens, b.starts)
        assert torch.equal(out, eager)
        full_k, full_v = b.keys, b.values
        b.keys, b.values = [k[:c + n] for k, c, n in zip(full_k, ctx, b.new)], [v[:c + n] for v, c, n in zip(full_v, ctx, b.new)]
        b.check(out)
        b.keys, b.values = full_k, full_v


def test_refusals():
    b = _Batch([10], [2], 4, 2, 64, 16, words=1)
    good = dict(q=b.q, k_pages=b.k, v_pages=b.v, tables=b.tables, lens=b.lens, starts=b.starts, masks=b.masks)
    gpuk.paged_attention(**good)
    wide = torch.zeros(2, 4, 65, dtype=torch.bfloat16, device="cuda")
    for more, text in [({"q": b.q.half()}, "types"), ({"q": b.q.float()}, "bfloat16 or float16"), ({"q": b.q[0]}, "tokens, heads"), ({"q": b.q.transpose(1, 2)}, "contiguous heads"),
                       ({"q": wide[..., 1:]}, "aligned|strides"), ({"k_pages": b.k.transpose(2, 3)}, "one size|contiguous"), ({"v_pages": b.v[:, :1]}, "one size"),
                       ({"v_pages": b.v.transpose(1, 2).contiguous().transpose(1, 2)}, "same strides"), ({"tables": b.tables.long()}, "int32"), ({"tables": b.tables[:0]}, "rows"),
                       ({"lens": b.lens.long()}, "lens"), ({"starts": b.starts[:1]}, "starts"), ({"masks": b.masks[:1]}, "masks"), ({"masks": torch.zeros(2, 9, dtype=torch.int32, device="cuda")}, "at most 8"),
                       ({"lens": b.lens.cpu()}, "CUDA"), ({"out": b.q}, "overlaps"), ({"out": torch.empty(2, 4, 32, dtype=torch.bfloat16, device="cuda")}, "size"),
                       ({"q": b.q.clone().requires_grad_()}, "gradient"), ({"q": b.q.expand(2, 4, 64)[:, :1].expand(2, 4, 64)}, "strides")]:
        with pytest.raises((RuntimeError, ValueError), match=text):
            gpuk.paged_attention(**{**good, **more})
    with torch.no_grad():
        gpuk.paged_attention(**{**good, "q": b.q.clone().requires_grad_()})
    # a plan writes nothing over what it reads
    ints = [_ints([3, 4]), _ints([1, 2]), _ints([[0, -1], [1, -1]]), _ints([1, 1]), _ints([2, 3, 0, 0]), _ints([2, 0])]
    for more, text in [({"held_out": ints[0]}, "overlap"), ({"free_count_out": ints[3]}, "overlap"), ({"held_out": ints[5], "free_count_out": ints[5]}, "overlap"),
                       ({"parents": _ints([0, 0, 0])}, "max_new"), ({"parents": _ints([0, 0, 0]), "max_new": 257}, "max_new"), ({"parents": _ints([0, 0]), "max_new": 2}, "parents")]:
        with pytest.raises(RuntimeError, match=text):
            gpuk.paged_plan(*ints, 16, 3, **more)
    with pytest.raises(RuntimeError, match="overlap"):
        gpuk.paged_plan(ints[0], ints[1], ints[2], ints[3], ints[2].view(-1), ints[5], 16, 3)
    with pytest.raises(RuntimeError, match="rows of tables"):
        gpuk.paged_plan(ints[0], ints[1], ints[2][:1].expand(2, 2), ints[3], ints[4], ints[5], 16, 3)
    with pytest.raises(RuntimeError, match="powers of two"):
        gpuk.paged_plan(*ints, 24, 3)
    x, pos, f = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda"), gpuk.rope_frequencies(64, device="cuda")
    for call, text in [(lambda: gpuk.rope(x, pos[:2], f), "positions"), (lambda: gpuk.rope(x, pos.int(), f), "positions"), (lambda: gpuk.rope(x, pos, f, out=x, layout="split"), "overlaps"),
                       (lambda: gpuk.rope(x[1:], pos[1:], f, out=x[:-1]), "overlaps"), (lambda: gpuk.rope(x[..., :48], pos, f), "rotated"),
                       (lambda: gpuk.rope(x, pos, gpuk.rope_frequencies(64)), "CUDA"), (lambda: gpuk.rope_paged(x, x, x, pos, pos, f, b.k, b.k[:, :1]), "one size"),
                       (lambda: gpuk.rope_paged(x, x[:, :1], x[:, :1], pos, pos, f, b.k, b.v), "shapes"), (lambda: gpuk.rope_paged(x, x, x, pos, pos, f, b.k.half(), b.v.half()), "one type"),
                       (lambda: gpuk.rope_paged(x, x, x, pos, pos[:1], f, b.k, b.v), "slots"), (lambda: gpuk.rope_paged(x, x, x, pos, pos, f, b.k, b.v, out=b.k[0, :, :3].transpose(0, 1)), "overlaps"),
                       (lambda: gpuk.paged_keep(b.k, b.k, b.tables, b.lens, _ints([[1]])), "overlap"), (lambda: gpuk.paged_keep(b.k, b.v, b.tables, b.lens, _ints([[1]]), out=b.lens), "overlaps"),
                       (lambda: gpuk.paged_keep(b.k, b.v, b.tables, b.lens, _ints([1])), "paths")]:
        with pytest.raises((RuntimeError, ValueError), match=text):
            call()
    torch.cuda.synchronize()


def test_empty_calls():
    """No requests, no tokens, nothing new: nothing is launched that reads anything."""
    b = _Batch([10, 0], [0, 0], 4, 2, 64, 16)
    assert b.run().shape == (0, 4, 64)
    none = _ints([])
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16, device="cuda")
    out = torch.full_like(q, 2.0)
    gpuk.paged_attention(q, b.k, b.v, none.view(0, 5), none, _ints([0]), out=out)
    gpuk.paged_attention(q, b.k, b.v, b.tables, b.lens, _ints([0, 0, 0]), out=out)
    assert bool((out == 2).all())
    f, pos = gpuk.rope_frequencies(64, device="cuda"), torch.zeros(0, dtype=torch.int64, device="cuda")
    assert gpuk.rope(q[:0], pos, f).shape == (0, 4, 64)
    gpuk.rope_paged(q[:0], q[:0, :2], q[:0, :2], pos, pos, f, b.k, b.v)
    assert gpuk.paged_keep(b.k, b.v, none.view(0, 5), none, none.view(0, 2)).shape == (0,)
    assert gpuk.paged_keep(b.k, b.v, b.tables, b.lens, none.view(2, 0)).tolist() == [10, 0]
    cabi.check(cabi.lib.gpuk_fp8_linear_status())
