"""The barriers of the attention over packed prompts, checked on the CPU.

Both kernels (speech-mac_b200/csrc/phonon_prompt.cuh) are agents that meet at barriers: copies or converters that fill
rings of keys and values, warps that issue products, the tensor cores that work products off in the order of their
issue, and softmax warps. Waits go by parity, so a waiter that lags two phases behind takes the phase before for the one
that it asks for, and one that is two phases early waits for good. The models below run the agents' waits and arrivals in
the kernels' order under random interleavings, with commits that arrive as late as they like and in any order, and say

- which waits could not tell the phase that they ask for from another,
- what was written while it was still to be read (a stage, a score tile, an output),
- whether every agent came to its end."""
import random

import pytest


class Bar:
    def __init__(self, count):
        self.count, self.pending, self.phases = count, count, 0

    def arrive(self):
        self.pending -= 1
        if self.pending == 0:
            self.phases, self.pending = self.phases + 1, self.count


class Run:
    """Agents are generators that yield whether they moved."""

    def __init__(self, seed, lag):
        self.rnd, self.lag, self.wrong, self.queue, self.late = random.Random(seed), lag, [], [], []

    def wait(self, bar, use, who):
        while bar.phases % 2 == use % 2:  # the phase of this parity is not the one before the present
            if bar.phases > use:
                self.wrong.append(f"{who}: waits for phase {use} again, {bar.phases} done")
                return
            yield False
        if bar.phases <= use:
            self.wrong.append(f"{who}: takes phase {bar.phases - 1} for {use}")
        yield True

    def tensor(self):
        """Products in the order of their issue; what a commit says arrives some time after."""
        while True:
            if self.queue:
                work, bars = self.queue.pop(0)
                work()
                self.late += bars
            yield bool(self.queue)

    def arrivals(self):
        while True:
            if self.late and self.rnd.random() < self.lag:
                self.late.pop(self.rnd.randrange(len(self.late))).arrive()
                yield True
            else:
                yield bool(self.late)

    def go(self, agents, paces):
        agents = agents + [self.tensor(), self.arrivals()]
        paces = paces + [self.rnd.choice([1, 0.1]), 1]
        left, idle = set(range(len(agents))), 0
        while any(a < len(agents) - 2 for a in left) and idle < 20000:
            order = sorted(left)
            who = self.rnd.choices(order, [paces[a] for a in order])[0]
            try:
                idle = 0 if next(agents[who]) else idle + 1
            except StopIteration:
                left.discard(who)
                idle = 0
        return self.wrong, not any(a < len(agents) - 2 for a in left)


def run_bf16(seed, stages, issuers, parts, ranges, lag, wait_for_scores=True):
    """ranges: of the two row tiles' turns."""
    r = Run(seed, lag)
    turns = max(e for _, e in ranges)
    ring = lambda count: [Bar(count) for _ in range(stages)]  # noqa: E731
    k_full, v_full, k_empty, v_empty = ring(1), ring(1), ring(issuers), ring(issuers)
    s_full, o_full = [Bar(1), Bar(1)], [Bar(1), Bar(1)]
    p_full = [[Bar(1) for _ in range(parts)] for _ in range(2)]
    k_at, v_at = [None] * stages, [None] * stages  # the turn that a stage holds
    todo_k, todo_v = {}, {}                        # products of a turn that have not read it
    s_at, read, summed = [None, None], [None, None], [-1, -1]

    def producer():
        for j in range(turns):
            s = j % stages
            for full, empty, at, todo, name in ((k_full, k_empty, k_at, todo_k, "keys"), (v_full, v_empty, v_at, todo_v, "values")):
                if j >= stages:
                    yield from r.wait(empty[s], j // stages - 1, f"producer, {name}")
                if at[s] is not None and todo.get(at[s]):
                    r.wrong.append(f"{name} of turn {at[s]} overwritten")
                at[s] = j
                todo[j] = {t for t, (b, e) in enumerate(ranges) if b <= j < e}
                r.late.append(full[s])  # the copy
                yield True

    def score(tile, j, last):
        b, e = ranges[tile]
        if b <= j < e:
            def work():
                if k_at[j % stages] != j:
                    r.wrong.append(f"S of turn {j} from other keys")
                todo_k[j].discard(tile)
                if j > b and summed[tile] != j - 1:
                    r.wrong.append(f"S of turn {j} over weights that are still to be read")
                s_at[tile] = j
            r.queue.append((work, [s_full[tile]]))
        if last:
            r.queue.append((lambda: None, [k_empty[j % stages]]))

    def sums(tile, j, last):
        b, e = ranges[tile]
        if b <= j < e:
            for h in range(parts):
                yield from r.wait(p_full[tile][h], j - b, f"issuer, weights of tile {tile}")

                def work(h=h):
                    if v_at[j % stages] != j or s_at[tile] != j:
                        r.wrong.append(f"P v of turn {j} from others")
                    if h == parts - 1:
                        todo_v[j].discard(tile)
                        summed[tile] = j
                r.queue.append((work, []))
            if j + 1 == e:
                r.queue.append((lambda: None, [o_full[tile]]))
        if last:
            r.queue.append((lambda: None, [v_empty[j % stages]]))

    def issuer(tiles):
        state = {"k": 0, "v": 0}

        def keys(j):
            if j >= state["k"]:
                yield from r.wait(k_full[j % stages], j // stages, "issuer, keys")
                state["k"] = j + 1

        def values(j):
            if j >= state["v"]:
                yield from r.wait(v_full[j % stages], j // stages, "issuer, values")
                state["v"] = j + 1
        for n, t in enumerate(tiles):
            yield from keys(0)
            score(t, 0, n + 1 == len(tiles))
        for j in range(turns):
            for n, t in enumerate(tiles):
                last = n + 1 == len(tiles)
                yield from values(j)
                if j + 1 < turns:
                    yield from keys(j + 1)
                yield from sums(t, j, last)
                if j + 1 < turns:
                    score(t, j + 1, last)
                yield True

    def softmax(tile):
        b, e = ranges[tile]
        for j in range(b, e):
            if wait_for_scores:
                yield from r.wait(s_full[tile], j - b, f"tile {tile}, scores")
            if s_at[tile] != j or (j > b and summed[tile] != j - 1):
                r.wrong.append(f"tile {tile} reads S or O of turn {j} too early")
            for h in range(parts):
                p_full[tile][h].arrive()
                yield True
        if e > b:
            yield from r.wait(o_full[tile], 0, f"tile {tile}, the end")
            if summed[tile] != e - 1:
                r.wrong.append(f"tile {tile} reads O before the last sum")

    agents = [producer()] + [issuer([0, 1])] * (issuers == 1) + ([issuer([0]), issuer([1])] if issuers == 2 else []) + [softmax(0), softmax(1)]
    return r.go(agents, [r.rnd.choice([1, 1, 0.3, 0.05]) for _ in agents])


def run_f32(seed, stages, buffers, parts, turns, lag, careful=False, rotate=4):
    r = Run(seed, lag)
    ring = lambda count: [Bar(count) for _ in range(stages)]  # noqa: E731
    k_full, v_full, k_empty, v_empty = ring(8), ring(8), ring(1), ring(1)
    s_full, o_full = [Bar(1) for _ in range(buffers)], [Bar(1) for _ in range(rotate)]
    p_full, q_full, meet = Bar(4), Bar(4), Bar(8)
    scored, summed = [False] * turns, [False] * turns
    taken = [0] * (turns + 1)   # warps that have added P v of a turn to their O
    read = [0] * turns          # warps that have S of a turn
    weighed = [0] * turns

    def converter():
        met = 0
        for n in range(turns * 2 * parts):
            values, j = n // parts & 1, n // (2 * parts)
            s = j % stages
            if n % parts == 0:
                if j >= stages:
                    yield from r.wait((v_empty if values else k_empty)[s], j // stages - 1, "converter")
                if careful:
                    if j >= stages:
                        yield from r.wait(v_empty[s], j // stages - 1, "converter, careful")
                    meet.arrive()
                    while meet.phases <= met:  # a named barrier: not by parity
                        yield False
                    met += 1
            if j >= stages and not (summed if values else scored)[j - stages]:
                r.wrong.append(f"stage of turn {j - stages} overwritten")
            if n % parts == parts - 1:
                (v_full if values else k_full)[s].arrive()
            yield True

    def score():
        yield from r.wait(q_full, 0, "score, q")
        for j in range(turns):
            if j >= buffers:
                yield from r.wait(o_full[(j - buffers) % rotate], (j - buffers) // rotate, "score, the sum before")
            yield from r.wait(k_full[j % stages], j // stages, "score, keys")

            def work(j=j):
                if j >= buffers and not summed[j - buffers]:
                    r.wrong.append(f"S of turn {j} over weights that are still to be read")
                scored[j] = True
            r.queue.append((work, [s_full[j % buffers], k_empty[j % stages]]))
            yield True

    def sums():
        for j in range(turns):
            yield from r.wait(v_full[j % stages], j // stages, "sum, values")
            yield from r.wait(p_full, j, "sum, weights")

            def work(j=j):
                if weighed[j] < 4 or (j and taken[j - 1] < 4):
                    r.wrong.append(f"P v of turn {j} too early")
                summed[j] = True
            r.queue.append((work, [o_full[j % rotate], v_empty[j % stages]]))
            yield True

    def softmax():
        q_full.arrive()

        def add(j):
            yield from r.wait(o_full[j % rotate], j // rotate, "softmax, the sum")
            if not summed[j]:
                r.wrong.append(f"O of turn {j} read before it is there")
            taken[j] += 1
        for j in range(turns):
            yield from r.wait(s_full[j % buffers], j // buffers, "softmax, scores")
            if not scored[j]:
                r.wrong.append(f"S of turn {j} read before it is there")
            if careful:
                yield from r.wait(k_full[j % stages], j // stages, "softmax, keys")
                yield from r.wait(v_full[j % stages], j // stages, "softmax, values")
            read[j] += 1
            weighed[j] += 1
            if j:
                yield from add(j - 1)
            p_full.arrive()
            yield True
        yield from add(turns - 1)

    agents = [converter() for _ in range(8)] + [score(), sums()] + [softmax() for _ in range(4)]
    return r.go(agents, [r.rnd.choice([1, 1, 0.3, 0.05]) for _ in agents])


RANGES = [((0, 1), (0, 0)), ((0, 1), (0, 1)), ((0, 5), (0, 6)), ((0, 12), (0, 12)), ((0, 9), (0, 0)), ((0, 3), (2, 5)), ((0, 2), (1, 3)),
          ((0, 17), (3, 18)), ((0, 2), (2, 4))]


@pytest.mark.parametrize("lag", [1.0, 0.2, 0.02])
@pytest.mark.parametrize("ranges", RANGES)
@pytest.mark.parametrize("stages,issuers,parts", [(2, 1, 2), (4, 2, 1)])  # 128 dims; up to 64
def test_bf16_kernel(stages, issuers, parts, ranges, lag):
    for seed in range(8):
        assert run_bf16(seed, stages, issuers, parts, ranges, lag) == ([], True)


@pytest.mark.parametrize("lag", [1.0, 0.2, 0.02])
@pytest.mark.parametrize("careful", [False, True])
@pytest.mark.parametrize("stages,buffers,parts", [(2, 2, 2), (3, 3, 1)])  # 128 dims; up to 64
def test_f32_kernel(stages, buffers, parts, careful, lag):
    for seed in range(6):
        for turns in (1, 2, 3, 7, 20):
            assert run_f32(seed, stages, buffers, parts, turns, lag, careful) == ([], True)


def test_the_models_see_what_they_are_there_for():
    """Scores read without a wait; and sums by one barrier, which a slow warp cannot tell apart."""
    assert any(run_bf16(seed, 4, 2, 1, ((0, 9), (0, 9)), 0.2, wait_for_scores=False)[0] for seed in range(5))
    bad = [run_f32(seed, 3, 3, 1, 30, 0.2, rotate=1) for seed in range(40)]
    assert any(wrong or not ended for wrong, ended in bad)
