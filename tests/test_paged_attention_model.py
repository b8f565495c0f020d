"""Host-side model of the paged attention kernel's roles (csrc/paged_attention.cu): copies, multiplications and row threads meet at mbarriers whose waits know only a parity.

Random interleavings: every wait has to see the phase that it means, nothing may be overwritten that is still read, everybody has to come to the end, and no
arrival may be left for behind it.  And the line of tiles that CTAs share: every block of every tile is taken once, and joined from the slots it was left in."""
import random

import pytest

QUEUE = 4


class Barrier:
    def __init__(self, arrivals):
        self.arrivals, self.left, self.phase, self.due = arrivals, arrivals, 0, 0

    def arrive(self):
        self.left -= 1
        assert self.left >= 0
        if self.left == 0:
            self.phase, self.left = self.phase + 1, self.arrivals

    def complete(self, parity):
        return (self.phase & 1) != parity


def _wait(barrier, index):
    """Waits as the kernel does, by the parity of phase `index`, and checks that it was that phase."""
    while not barrier.complete(index & 1):
        yield False
    assert barrier.phase == index + 1, (barrier.phase, index)


def _run(segments, slots, warps, rng, rescales, masked):
    full, empty = [Barrier(1) for _ in range(slots)], [Barrier(1) for _ in range(slots)]
    q_full, s_full, o_done, p_full = ([Barrier(n) for _ in range(2)] for n in (1, 1, 1, warps))
    q_empty, together = Barrier(1), Barrier(warps)
    queue, copies, tensor = [None] * QUEUE, [], []
    q_held, ring, scores_done, product_done = [None], [None] * slots, [-1], [-1]
    reading_ring, reading_queue = [0] * slots, [0] * QUEUE

    def copier():
        filled = 0
        for number, blocks in enumerate(segments):
            def load(what):
                nonlocal filled
                slot = filled % slots
                if filled >= slots:
                    yield from _wait(empty[slot], filled // slots - 1)
                else:
                    assert empty[slot].complete(1)
                assert not reading_ring[slot]
                copies.append((slot, what))
                filled += 1
                yield True
            yield from load(("k", number, 0))
            if number:
                yield from _wait(q_empty, number - 1)
            assert not reading_queue[number % QUEUE]
            queue[number % QUEUE] = (number, blocks)
            copies.append(("q", number))
            for j in range(blocks):
                if j + 1 < blocks:
                    yield from load(("k", number, j + 1))
                yield from load(("v", number, j))
        yield from _wait(q_empty, len(segments) - 1)
        assert not reading_queue[len(segments) % QUEUE]
        queue[len(segments) % QUEUE] = (len(segments), 0)
        q_full[len(segments) & 1].arrive()
        for i in range(max(0, filled - slots), filled):
            yield from _wait(empty[i % slots], i // slots)

    def multiplier():
        fill = t = number = 0
        while True:
            yield from _wait(q_full[number & 1], number >> 1)
            got, blocks = queue[number % QUEUE]
            assert got == number
            if not blocks:
                return

            def scores(t, i, j):
                tensor.append(("s", t, number, j, i % slots))
                tensor.append(s_full[t & 1])
                tensor.append(empty[i % slots])
                if j + 1 == blocks:
                    tensor.append(q_empty)
            yield from _wait(full[fill % slots], fill // slots)
            scores(t, fill, 0)
            for j in range(blocks):
                if j + 1 < blocks:
                    i = fill + 2 * j + 1
                    yield from _wait(full[i % slots], i // slots)
                    scores(t + 1, i, j + 1)
                i = fill + (2 * j + 2 if j + 1 < blocks else 2 * j + 1)
                yield from _wait(full[i % slots], i // slots)
                yield from _wait(p_full[t & 1], t >> 1)
                tensor.append(("o", t, number, j, i % slots))
                tensor.append(empty[i % slots])
                tensor.append(o_done[t & 1])
                t += 1
                yield True
            fill += 2 * blocks
            number += 1

    def rows(_):
        t = fill = number = 0
        while True:
            yield from _wait(q_full[number & 1], number >> 1)
            reading_queue[number % QUEUE] += 1
            got, blocks = queue[number % QUEUE]
            assert got == number
            yield True
            assert queue[number % QUEUE] == (got, blocks)
            reading_queue[number % QUEUE] -= 1
            if not blocks:
                break
            for j in range(blocks):
                yield from _wait(s_full[t & 1], t >> 1)
                assert scores_done[0] in (t, t + 1)
                if j and rescales():
                    yield from _wait(o_done[(t - 1) & 1], (t - 1) >> 1)
                    assert product_done[0] == t - 1
                yield True
                if masked():
                    i = fill + (2 * j + 2 if j + 1 < blocks else 2 * j + 1)
                    yield from _wait(full[i % slots], i // slots)
                    assert ring[i % slots] == ("v", number, j)
                    reading_ring[i % slots] += 1
                    yield True
                    reading_ring[i % slots] -= 1
                p_full[t & 1].arrive()
                t += 1
            fill += 2 * blocks
            yield from _wait(o_done[(t - 1) & 1], (t - 1) >> 1)
            assert product_done[0] == t - 1
            together.arrive()
            yield from _wait(together, number)
            yield True
            assert product_done[0] == t - 1      # the outputs stay while they are read
            number += 1
        if t > 1:
            yield from _wait(o_done[t & 1], (t - 2) >> 1)

    def hardware():
        if copies and rng.random() < 0.5:
            at, *what = copies.pop(rng.randrange(min(2, len(copies))))
            if at == "q":
                q_held[0] = what[0]
                q_full[what[0] & 1].arrive()
            else:
                ring[at] = what[0]
                full[at].arrive()
        if tensor and rng.random() < 0.6:
            op = tensor.pop(0)
            if isinstance(op, Barrier):
                op.arrive()
                return
            kind, t, number, j, slot = op
            assert ring[slot] == ("k" if kind == "s" else "v", number, j)
            if kind == "s":
                assert q_held[0] == number
                scores_done[0] = t
            else:
                product_done[0] = t

    roles = [copier(), multiplier()] + [rows(w) for w in range(warps)]
    bias, idle = rng.choice([0.0, 0.5, 0.9]), 0
    while roles:
        hardware()
        role = roles[0] if rng.random() < bias else rng.choice(roles)
        for _ in range(rng.choice([1, 2, 8])):
            try:
                idle = 0 if next(role) else idle + 1
            except StopIteration:
                roles.remove(role)
                idle = 0
                break
        assert idle < 100000, "a wait that never ends"
    assert not copies and not tensor, "something arrives behind the end"


@pytest.mark.parametrize("slots", [5, 10])
def test_roles_meet(slots):
    rng = random.Random(slots)
    for _ in range(500):
        segments = [rng.choice([1, 1, 2, 3, 4, 5, 9]) for _ in range(rng.choice([1, 2, 3, 6]))]
        often, mask = rng.choice([0.0, 0.2, 1.0]), rng.choice([0.0, 0.3, 1.0])
        _run(segments, slots, 4, rng, lambda: rng.random() < often, lambda: rng.random() < mask)


# ---- the line of tiles ------------------------------------------------------------------------------------------------
KEYS, COST, FRONT, GRAIN, PER_CTA, SMALL = 64, 256, 192, 128, 256, 6


def _share(requests, kv_heads, tile_tokens, masks, room, grid, may_split=True):
    """Segments (tile, first, last, slot) of each CTA, as find_start and Walk of the kernel give them."""
    reqs = []
    for ctx, n in requests:
        ctx = min(ctx, room)
        reqs.append((ctx, n, -(-n // tile_tokens), ctx + n > room))

    def before(r, tile):
        ctx, n, tiles, over = r
        if tiles == 0:
            return 0
        if masks or over:
            return tile * (COST + min(ctx + n, room))
        whole = min(tile, tiles - 1)
        w = whole * (COST + ctx) + tile_tokens * (whole * (whole + 1) // 2)
        return w if tile < tiles or tile == 0 else w + COST + ctx + n

    def keys(r, tile):
        ctx, n, _, _ = r
        return min(ctx + (n if masks else min(n, (tile + 1) * tile_tokens)), room)

    total = sum(before(r, r[2]) * kv_heads for r in reqs)
    few = sum(r[2] for r in reqs) * kv_heads
    ctas = max(1, min(grid, 2 * few + total // PER_CTA))
    share = int(total * 1.00001 / ctas) + 1
    largest = max(before(r, r[2]) - before(r, r[2] - 1) for r in reqs if r[2])
    may_split = may_split and not (few <= grid and 2 * largest <= 3 * share) and SMALL * largest > share

    def border(c):
        raw, base = min(total, c * share), 0
        for i, r in enumerate(reqs):
            head = before(r, r[2])
            if raw >= base + head * kv_heads:
                base += head * kv_heads
                continue
            kvh = (raw - base) // head
            at = raw - base - kvh * head
            tile = max(k for k in range(r[2]) if before(r, k) <= at)
            first, last = before(r, tile), before(r, tile + 1)
            pos = at - first
            if not may_split or r[3] or pos < COST + FRONT:
                pos = 0
            elif last - first - pos < GRAIN:
                pos = last - first
            else:
                pos = pos // KEYS * KEYS
            return base + kvh * head + first + pos, (i, kvh, tile, pos)
        return total, None

    out = []
    for c in range(ctas):
        (x0, at), (x1, _) = border(c), border(c + 1)
        left, mine, index = x1 - x0, [], 0
        if left > 0:
            i, kvh, tile, pos = at
        while left > 0:
            r = reqs[i]
            size = before(r, tile + 1) - before(r, tile)
            while pos >= size:
                pos, tile = 0, tile + 1
                if tile >= r[2]:
                    tile, kvh = 0, kvh + 1
                    if kvh >= kv_heads:
                        kvh, i = 0, i + 1
                        while reqs[i][2] == 0:
                            i += 1
                        r = reqs[i]
                size = before(r, tile + 1) - before(r, tile)
            take = min(size - pos, left)
            end, every = pos + take, -(-keys(r, tile) // KEYS)
            block = lambda w: 0 if w <= COST else min(-(-(w - COST) // KEYS), every)  # noqa: E731
            first, last = 0 if pos == 0 else block(pos), every if end == size else block(end)
            whole = pos == 0 and end == size
            mine.append(((i, kvh, tile), first, last, every, -1 if whole else 2 * c + (pos == 0 and index > 0), pos == 0, end == size))
            pos, left, index = end, left - take, index + 1
        out.append(mine)
    return reqs, out


@pytest.mark.parametrize("masks", [False, True])
def test_every_block_is_taken_once_and_found_again(masks):
    rng = random.Random(masks)
    for _ in range(300):
        batch, kv, tt = rng.choice([1, 2, 5, 40]), rng.choice([1, 3, 8]), rng.choice([1, 16, 25, 128])
        longest = rng.choice([10, 400, 3000, 20000])
        requests = [(rng.choice([0, rng.randint(0, longest)]), rng.choice([0, 1, 1, rng.randint(0, 70), rng.randint(0, 300)])) for _ in range(batch)]
        room = rng.choice([1 << 20, 1 << 20, longest // 2 + 8])
        if not any(n for _, n in requests):
            continue
        reqs, ctas = _share(requests, kv, tt, masks, room, rng.choice([1, 7, 296]), rng.random() < 0.9)
        taken, slots = {}, {}
        for c, mine in enumerate(ctas):
            for number, (tile, first, last, every, slot, begins, ends) in enumerate(mine):
                assert 0 <= first < last <= every
                taken.setdefault(tile, []).append((first, last, every))
                if slot >= 0:
                    assert slot not in slots and slot // 2 == c and (begins or number == 0) and not (begins and ends)
                    slots[slot] = tile
        expected = {(i, h, t) for i, r in enumerate(reqs) for h in range(kv) for t in range(r[2])}
        assert set(taken) == expected
        for pieces in taken.values():      # in order, without a gap
            assert pieces[0][0] == 0 and pieces[-1][1] == pieces[-1][2] and all(a[1] == b[0] for a, b in zip(pieces, pieces[1:]))
        # the second kernel's search: from the CTA where a tile begins to the one where it ends
        heads = [0 if not m else 3 if m[0][5] else 2 if m[0][6] else 1 for m in ctas]
        joined = {}
        for c, mine in enumerate(ctas):
            if mine and mine[-1][5] and not mine[-1][6]:
                parts = [mine[-1][4]]
                for d in range(c + 1, len(ctas)):
                    if heads[d] in (1, 2):
                        parts.append(2 * d)
                    if heads[d] >= 2:
                        break
                joined[mine[-1][0]] = parts
        assert sorted(s for parts in joined.values() for s in parts) == sorted(slots)
        assert all(slots[s] == tile for tile, parts in joined.items() for s in parts)
