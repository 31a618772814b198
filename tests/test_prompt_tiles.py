"""How a CTA of the attention over packed prompts finds its rows (prompt_find in speech-mac_b200/csrc/phonon_prompt.cuh),
and how many CTAs a call has, on the CPU: every position of every good prompt is one CTA's, no other row is anyone's, and
a prompt that has to be reported is seen by the CTAs of the last slot."""
import numpy as np
import pytest


def slots(rows, prompts, max_rows, tokens):
    """prompt_ctas, for one group of heads."""
    return min(rows // tokens + prompts, prompts * -(-max_rows // tokens))


def find(begin, rows, max_rows, tokens, slot):
    """(tile or none, prompts found bad): 128 prompts at a time, four a lane."""
    prompts = len(begin) - 1
    before = most = 0
    bad = []
    for base in range(0, prompts, 128):
        found, highest = None, []
        sums = 0
        run = most  # the largest begin so far, as the lanes' scan has it
        for lane in range(32):
            i = base + 4 * lane
            x = [begin[min(i + k, prompts)] for k in range(5)]
            for k in range(4):
                b, e = x[k], x[k + 1]
                good = b >= run and e >= b and e <= rows and e - b <= max_rows
                tiles = 0
                if i + k < prompts:
                    if not good:
                        bad.append(i + k)
                    else:
                        tiles = (e - b + tokens - 1) // tokens
                at = slot - (before + sums)
                if 0 <= at < tiles:
                    found = (i + k, b, e - b, (tiles - 1 - at) * tokens)
                sums += tiles
                run = max(run, b)
            highest.append(max(x[:4]))
        before += sums
        most = max([most] + highest)
        if slot < before:
            return found, bad
    return None, bad


def check(begin, rows, max_rows, tokens):
    n = slots(rows, len(begin) - 1, max_rows, tokens)
    owner = np.zeros(rows, int)
    for s in range(n):
        tile, bad = find(begin, rows, max_rows, tokens, s)
        if tile:
            i, row0, length, first = tile
            assert 0 <= row0 and row0 + length <= rows and 0 <= first < length
            owner[row0 + first:row0 + min(length, first + tokens)] += 1
    want, top, wrong = np.zeros(rows, int), 0, []
    for i, (b, e) in enumerate(zip(begin, begin[1:])):
        if b >= top and b <= e <= rows and e - b <= max_rows and b >= 0:
            want[b:e] += 1
        else:
            wrong.append(i)
        top = max(top, b)
    assert (want <= 1).all() and (owner == want).all()
    if wrong:
        assert tile is None and bad == wrong  # of the last slot


@pytest.mark.parametrize("tokens", [1, 3, 128, 256])
@pytest.mark.parametrize("prompts", [1, 4, 5, 127, 128, 129, 300])
def test_every_row_once(tokens, prompts):
    rng = np.random.default_rng(tokens + prompts)
    for most in (1, tokens, 3 * tokens):
        for empty in (0.0, 0.5, 0.9):
            lengths = rng.integers(1, most + 1, prompts) * (rng.random(prompts) >= empty)
            begin = np.concatenate([[0], np.cumsum(lengths)]) + rng.integers(0, 3)
            rows = max(1, int(begin[-1]) + int(rng.integers(0, 3)))
            check([int(b) for b in begin], rows, max(1, min(rows, int(lengths.max()))), tokens)
            check([int(b) for b in begin], rows, rows, tokens)


@pytest.mark.parametrize("prompts", [1, 3, 130, 260])
def test_bad_prompts_have_no_tile_and_are_reported(prompts):
    rng = np.random.default_rng(prompts)
    for _ in range(20):
        lengths = rng.integers(0, 9, prompts)
        begin = np.concatenate([[0], np.cumsum(lengths)])
        rows = max(1, int(begin[-1]))
        for _ in range(rng.integers(1, 4)):
            begin[rng.integers(0, prompts + 1)] = rng.choice([-5, 0, rows // 2, rows, rows + 1, 2 ** 31 - 1, -2 ** 31])
        check([int(b) for b in begin], rows, min(rows, int(rng.integers(1, 9))), 4)
