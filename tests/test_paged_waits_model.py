"""Host-side model of waits that give up in the paged attention kernel (csrc/paged_attention.cu): lanes with clocks of their own, and what only whole warps can do.

A wait on an mbarrier gives up after a while.  What follows it (shuffles, loads of tensor memory, __syncwarp) is for the whole warp, so all lanes have to go on from it alike: they go on as if it were over,
and from one segment to the next by a vote.  Completions come late here, some after a lane's patience and before another's: everybody has to come to the end soon, no warp may be torn, and nothing
that was issued may be in flight when shared and tensor memory are given back."""
import os
import random
import re

import pytest

from tests.test_paged_attention_model import QUEUE, Barrier

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gpuk_b200", "csrc")
LANES, ROW_WARPS = 2, 2


class Torn(Exception):
    """Lanes of a warp at different collective instructions, or one that never ends."""


def _run(segments, slots, rng, together_on):
    full, empty = [Barrier(1) for _ in range(slots)], [Barrier(1) for _ in range(slots)]
    q_full, s_full, o_done, p_full = ([Barrier(n) for _ in range(2)] for n in (1, 1, 1, ROW_WARPS))
    q_empty, together, drained = Barrier(1), Barrier(ROW_WARPS), Barrier(1)
    queue, copies, tensor = [None] * QUEUE, [], []
    # how long each completion takes: mostly at once, now and then about as long as the waits, or far longer
    late = lambda: rng.choice([0] * 40 + [rng.randint(50, 120), rng.randint(400, 2000)])  # noqa: E731
    gave_up = [False]

    def lane_wait(barrier, index, patience, alone=False):
        spins = 0
        while not barrier.complete(index & 1):
            spins += 1
            if spins > patience or (together_on and not alone and gave_up[0] and spins > 3):
                gave_up[0] = True
                return False
            yield None
        return True

    def make_wait():
        patience = rng.randint(60, 100)
        return lambda barrier, index: lane_wait(barrier, index, patience)

    def vote(ok):
        if together_on:
            ok = yield ("vote", ok)
        return ok

    def copier(lane):
        wait, ok, filled, number = make_wait(), True, 0, 0

        def load(ok, index):
            if ok or together_on:
                there = yield from wait(empty[index % slots], index // slots - 1 if index >= slots else 1)
                ok = ok and there
            if not ok and not together_on:
                return False
            yield ("expect", True)
            if lane == 0 and ok:
                copies.append([late(), full[index % slots]])
            return ok

        def load_q(blocks):
            if lane == 0:
                queue[number % QUEUE] = (number, blocks)
                copies.append([late(), q_full[number & 1]])

        for blocks in segments:
            yield ("pages", True)
            if number == 0:
                load_q(blocks)
            ok = yield from load(ok, filled)
            filled += ok
            if number > 0:
                there = yield from wait(q_empty, number - 1)
                ok = yield from vote(ok and there and (not together_on or not gave_up[0]))
                if not ok:
                    break
                load_q(blocks)
            number += 1
            for j in range(blocks):
                if j + 1 < blocks and (ok or together_on):
                    yield ("next page", True)
                    ok = yield from load(ok, filled)
                    filled += ok
                if ok or together_on:
                    ok = yield from load(ok, filled)
                    filled += ok
            ok = yield from vote(ok)
            if not ok:
                break
        if ok and number > 0:
            ok = yield from wait(q_empty, number - 1)
        if ok and lane == 0:
            queue[number % QUEUE] = (number, 0)
            q_full[number & 1].arrive()
        if not ok and number > 0:
            yield from lane_wait(q_full[(number - 1) & 1], (number - 1) >> 1, 3000, True)
        for i in range(max(0, filled - slots), filled):
            if ok:
                ok = yield from wait(empty[i % slots], i // slots)
            if not ok:
                landed = yield from lane_wait(full[i % slots], i // slots, 3000, True)
                if not landed:
                    break

    def multiplier(lane):
        own, fill, t, number = make_wait(), 0, 0, 0

        def wait(barrier, index):      # this warp votes behind each
            ok = yield from own(barrier, index)
            ok = yield from vote(ok)
            return ok

        def issue(*arrivals):
            if lane == 0:
                tensor.append(late())
                tensor.extend(arrivals)

        def scores(last):
            issue(s_full[t & 1], empty[fill % slots], *([q_empty] if last else []))

        ok = True
        while ok:
            ok = yield from wait(q_full[number & 1], number >> 1)
            if not ok:
                break
            got, blocks = yield ("blocks", queue[number % QUEUE])
            assert got == number or not together_on
            if not blocks:
                break
            ok = yield from wait(full[fill % slots], fill // slots)
            if ok:
                yield ("elect", True)
                scores(blocks == 1)
                fill += 1
            for j in range(blocks):
                if not ok:
                    break
                if j + 1 < blocks:
                    ok = yield from wait(full[fill % slots], fill // slots)
                    if not ok:
                        break
                    yield ("elect", True)
                    t += 1
                    scores(j + 2 == blocks)
                    t -= 1
                    fill += 1
                ok = yield from wait(full[fill % slots], fill // slots)
                if ok:
                    ok = yield from wait(p_full[t & 1], t >> 1)
                if not ok:
                    break
                yield ("elect", True)
                issue(o_done[t & 1], empty[fill % slots])
                fill += 1
                t += 1
            number += 1
        yield ("elect", True)
        issue(drained)
        yield from lane_wait(drained, 0, 50000, True)

    def rows(lane):
        wait, t, fill, number, ok = make_wait(), 0, 0, 0, True
        masked = random.Random(len(segments)).random() < 0.5
        while ok:
            ok = yield from wait(q_full[number & 1], number >> 1)
            ok = yield from vote(ok and (not together_on or not gave_up[0]))
            if not ok:
                break
            got, blocks = queue[number % QUEUE]
            assert got == number or not together_on      # what a row's place in the outputs is computed from
            if not blocks:
                break
            for j in range(blocks):
                if not ok and not together_on:
                    break
                there = yield from wait(s_full[t & 1], t >> 1)
                ok = ok and there
                yield ("load of scores", True)
                if j:
                    there = yield from wait(o_done[(t - 1) & 1], (t - 1) >> 1)
                    ok = ok and there
                    yield ("load of outputs", True)
                if masked:
                    i = fill + (2 * j + 2 if j + 1 < blocks else 2 * j + 1)
                    there = yield from wait(full[i % slots], i // slots)
                    ok = ok and there
                yield ("arrival", True)
                if lane == 0:
                    p_full[t & 1].arrive()
                t += 1
            fill += 2 * blocks
            if ok or together_on:
                there = yield from wait(o_done[(t - 1) & 1], (t - 1) >> 1)
                ok = ok and there
            yield ("arrival at the end", True)
            if lane == 0:
                together.arrive()
            if ok or together_on:
                there = yield from wait(together, number)
                ok = ok and there
            yield ("outputs", True)
            number += 1
            if together_on:
                ok = True      # the vote of the next segment says
        if t > 1:
            yield from wait(o_done[t & 1], (t - 2) >> 1)

    def hardware():
        for c in list(copies):
            c[0] -= 1
            if c[0] < 0:
                copies.remove(c)
                c[1].arrive()
        # what is issued to the tensor core completes in order
        if tensor and isinstance(tensor[0], int):
            tensor[0] -= 1
            if tensor[0] < 0:
                tensor.pop(0)
        while tensor and not isinstance(tensor[0], int):
            tensor.pop(0).arrive()

    warps = [[role(lane) for lane in range(LANES)] for role in [copier, multiplier] + [rows] * ROW_WARPS]
    parked = [[None] * LANES for _ in warps]
    done = [[False] * LANES for _ in warps]
    for step in range(60000):
        if all(map(all, done)):
            break
        hardware()
        for w, warp in enumerate(warps):
            for lane, role in enumerate(warp):
                if done[w][lane] or parked[w][lane] or rng.random() < 0.3:
                    continue
                try:
                    parked[w][lane] = next(role)
                except StopIteration:
                    done[w][lane] = True
            if any(parked[w]) and all(p or d for p, d in zip(parked[w], done[w])):
                if any(done[w]) or len({p[0] for p in parked[w]}) > 1:
                    raise Torn([p and p[0] for p in parked[w]])
                value = all(p[1] for p in parked[w]) if parked[w][0][0] == "vote" else parked[w][0][1]
                for lane, role in enumerate(warp):
                    parked[w][lane] = None
                    try:
                        parked[w][lane] = role.send(value)
                    except StopIteration:
                        done[w][lane] = True
    else:
        raise Torn("somebody never ends")
    assert not tensor and not copies, "something is in flight at the end"
    return gave_up[0]


def test_warps_that_go_together_come_to_the_end():
    rng, times = random.Random(1), 0
    for _ in range(250):
        times += _run([rng.choice([1, 1, 2, 3, 5]) for _ in range(rng.choice([1, 2, 4]))], rng.choice([5, 10]), rng, True)
    assert times > 50      # runs in which a wait did give up


def test_lanes_that_go_alone_are_torn():
    """Why: each lane leaves its loops by its own verdict here."""
    rng, torn = random.Random(1), 0
    for _ in range(250):
        try:
            _run([rng.choice([1, 1, 2, 3, 5]) for _ in range(rng.choice([1, 2, 4]))], rng.choice([5, 10]), rng, False)
        except Torn:
            torn += 1
    assert torn > 10


def _section(source, begin, end):
    return source[source.index(begin):source.index(end)]


def test_what_the_kernel_does_about_it():
    """Inside a segment no branch, loop or way out is a lane's own affair; between segments and in the multiplying warp there is a vote; what was issued has come before memory is given back."""
    source = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, "paged_attention.cu")).read())
    copier, multiplier, rows, end = "if (warp == kRows / 32 + 1) {", "} else if (warp == kRows / 32) {", "int row_tok = tid / p.group", "if (tid == 0 && !(aligned && all_well())) *p.status = 1;"
    assert "return __all_sync(0xffffffffu, ok) != 0" in source and "return vote(wait(bar, parity))" in source
    for begin, stop in ((copier, multiplier), (rows, end)):
        code = _section(source, begin, stop)
        assert re.findall(r"for \(int j = 0;([^;]*);", code) == [" j < u.blocks"]
        body = code[code.index("for (int j = 0; j < u.blocks"):]
        body = re.sub(r"\[&\]\([^)]*\) \{[^}]*\}", "", body[:body.index("ok = vote(ok)" if begin == copier else "arrive_at(smem_addr(&sm.together))")])
        assert not re.search(r"\b(break|return|continue|ok)\b", body)
    assert re.findall(r"vote\([^;]*all_well\(\)\)", _section(source, rows, end)) and re.findall(r"vote\([^;]*all_well\(\)\)", _section(source, copier, multiplier))
    body = re.sub(r"auto wait_all = [^\n]*", "", _section(source, multiplier, rows))
    assert not re.search(r"[^_\w]wait\(", body)
    # a value is looked up again only in a page that is there, whatever a slot held that was not waited for
    assert re.search(r"page = p\.tables\[[^;]*;\s*if \(page < 0 \|\| page >= p\.num_pages\) continue;", _section(source, rows, end))
    assert source.count("tc_commit(&sm.drained)") == 1 and not re.search(r"if \(!ok\)\s*\{?\s*(if \(elect_one\(\)\) )?tc_commit\(&sm.drained\)", source)
