"""The paged cache at its edges, as far as it needs no GPU: rotary frequencies at the ends of their ramps, and callers that want to see what is computed."""
import math

import pytest
import torch

import gpuk_b200 as gpuk


# ---- rotary frequencies --------------------------------------------------------------------------------------
def _yarn(rotary, theta, factor, low, high, original):
    """From the definition: a ramp from 0 to 1 along the pairs, between the whole numbers around those that turn `high` and `low` times over the original context, clamped to the values of a
    head and not to its pairs; 1 is divided by the factor, 0 is left."""
    pair = lambda turns: rotary * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
    first, last = max(math.floor(pair(high)), 0), min(math.ceil(pair(low)), rotary - 1)
    out = []
    for i in range(rotary // 2):
        f, ramp = theta ** (-2 * i / rotary), min(max((i - first) / max(last - first, 0.001), 0.0), 1.0)
        out.append(f * (1 - ramp) + f / factor * ramp)
    return out


@pytest.mark.parametrize("rotary,theta,original,low,high", [(16, 10000.0, 32768, 1.0, 32.0), (16, 10000.0, 1 << 20, 1.0, 32.0), (32, 10000.0, 131072, 0.5, 64.0), (128, 500000.0, 4096, 1.0, 32.0),
                                                           (128, 100.0, 8192, 1.0, 32.0), (64, 10000.0, 100, 1.0, 32.0)])
def test_yarn_beyond_the_last_pair(rotary, theta, original, low, high):
    """The ramp ends where a pair would turn `low` times, be it beyond the last: pairs that turn more often are never divided by the whole factor."""
    f, amplitude = gpuk.paged.scaled_frequencies(rotary, theta, {"kind": "yarn", "factor": 16.0, "low": low, "high": high, "original": original})
    want = _yarn(rotary, theta, 16.0, low, high, original)
    # a few roundings of 64-bit numbers
    assert all(abs(a - b) <= 2.0 ** -50 * b for a, b in zip(f.tolist(), want))
    for i, x in enumerate(f.tolist()):
        plain = theta ** (-2 * i / rotary)
        if original * plain / (2 * math.pi) > low:
            assert x > plain / 16.0 * (1 + 2.0 ** -40)
    assert amplitude == 0.1 * math.log(16.0) + 1


def test_the_last_pair_of_a_short_head():
    """rotary 16, theta 10000, trained over 32768: the last pair turns 1.65 times, between the ramp's ends 4 and 8, and keeps 1/4 of its own and 3/4 of a sixteenth of its frequency."""
    f, _ = gpuk.paged.scaled_frequencies(16, 10000.0, {"kind": "yarn", "factor": 16.0, "low": 1.0, "high": 32.0, "original": 32768})
    assert math.isclose(float(f[7]), 10000.0 ** (-14 / 16) * (0.25 + 0.75 / 16), rel_tol=1e-14)


@pytest.mark.parametrize("factor", [0.5, 1.0])
def test_a_context_that_does_not_grow_keeps_its_amplitude(factor):
    _, amplitude = gpuk.paged.scaled_frequencies(64, 10000.0, {"kind": "yarn", "factor": factor, "low": 1.0, "high": 32.0, "original": 4096})
    assert amplitude == 1.0


# ---- callers that want to see what is computed ------------------------------------------------------------------
def test_modes_are_refused_first():
    """Before the arguments are looked at, by each of the calls."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    x, f = torch.zeros(3, 2, 64), gpuk.rope_frequencies(64)
    for call in (lambda: gpuk.paged_plan(x, x, x, x, x, x, 16, 3), lambda: gpuk.rope(x, x, f), lambda: gpuk.rope_paged(x, x, x, x, x, f, x, x),
                 lambda: gpuk.paged_attention(x, x, x, x, x, x), lambda: gpuk.paged_keep(x, x, x, x, x)):
        with pytest.raises(RuntimeError, match="dispatch mode"), Watch():
            call()
        with pytest.raises(RuntimeError, match="dispatch mode"):
            torch.func.vmap(lambda y: call())(torch.zeros(2, 1))
        with pytest.raises(RuntimeError, match="CUDA tensor"), torch.device("cpu"):      # a function mode
            call()


# ---- clusters that have no place ------------------------------------------------------------------------------
def test_the_cap_on_a_plan_s_cluster():
    from gpuk_b200 import cabi

    for value, status in ((16, cabi.OK), (1, cabi.OK), (0, cabi.OK), (3, cabi.ERR_INVALID_ARGUMENT), (32, cabi.ERR_INVALID_ARGUMENT), (-1, cabi.ERR_INVALID_ARGUMENT)):
        assert cabi.lib.gpuk_set_tuning(b"paged_plan_ctas", value) == status


# ---- caches that attention cannot read ------------------------------------------------------------------------
@pytest.mark.parametrize("more,text", [({"page_size": 4}, "pages of 4"), ({"page_size": 48}, "pages of 48"), ({"page_size": 1 << 17}, "pages of 131072"), ({"head_dim": 96}, "heads of 96"),
                                       ({"head_dim": 256}, "heads of 256"), ({"requests": 4097}, "4097 requests"), ({"dtype": torch.float32}, "bfloat16 or float16"), ({"kv_heads": 0}, "kv_heads"),
                                       ({"pages_per_request": 1 << 27}, "pages_per_request"), ({"layers": 0}, "layers=0"), ({"pages": 0}, "pages=0"), ({"pages_per_request": 0}, "pages_per_request=0"), ({"requests": -1}, "requests")])
def test_a_cache_is_refused_when_it_is_made(more, text):
    """Not by the first attention over it, when a plan has dealt out pages and a layer's keys are written."""
    good = dict(layers=1, pages=2, page_size=16, kv_heads=2, head_dim=64, requests=3, pages_per_request=2, dtype=torch.float16, device="cpu")
    gpuk.PagedKVCache(**good)
    with pytest.raises(ValueError, match=text):
        gpuk.PagedKVCache(**{**good, **more})


@pytest.mark.parametrize("more,text", [({"head_dim": 96}, "heads of 96"), ({"head_dim": 32}, "heads of 32"), ({"dtype": torch.float32}, "bfloat16 or float16"), ({"n_heads": 6, "n_kv_heads": 4}, "6 query heads"),
                                       ({"n_heads": 129, "n_kv_heads": 1}, "129 query heads")])
def test_a_decoder_refuses_a_cache_that_it_could_not_read(more, text):
    from gpuk_b200.tp_model import DecoderArgs, TPDecoder

    class Alone:
        rank, world_size = 0, 1

    def decoder(**more):
        return TPDecoder(DecoderArgs(**{**dict(dim=64, n_layers=1, n_heads=2, n_kv_heads=1, head_dim=64, ffn_dim=64, vocab_size=32, max_seq_len=16), **more}), Alone(), device="cpu", fp8=False, max_batch=1)

    assert decoder().paged_cache(4, 2, 2).page_size == 64
    with pytest.raises(ValueError, match=text):
        decoder(**more).paged_cache(4, 2, 2)
    with pytest.raises(ValueError, match="pages of 2"):
        decoder().paged_cache(4, 2, 2, page_size=2)


def test_masks_of_no_tokens_need_no_parents():
    """As far as the call looks at its arguments: with too many requests it goes no further."""
    from gpuk_b200 import cabi
    from tests.test_paged_host import P, _plan

    for parents, masks in ((None, P), (P, None), (None, None), (P, P)):
        assert _plan(total=0, parents=parents, masks=masks, words=1, positions=None, slots=None, free=None) == cabi.ERR_INVALID_ARGUMENT and "null" in cabi.last_error()
        if not parents != (not masks):
            assert _plan(total=1, parents=parents, masks=masks, words=1) == cabi.ERR_INVALID_ARGUMENT and "masks" in cabi.last_error()
