"""The cases of perf/more_operators.py, listed and drawn, through the framework's calls, against that file's definitions in 64
bits, and its plain forms beside them."""
import importlib.util
import random
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

PATH = Path(__file__).resolve().parent.parent / "perf" / "more_operators.py"
SPEC = importlib.util.spec_from_file_location("more_operators", PATH)
mo = importlib.util.module_from_spec(SPEC)
SPEC.loader.exec_module(mo)


def outputs(case, seed, own):
    mo.own = own
    try:
        y = mo.run(mo.prepare(case, seed))
        torch.cuda.synchronize()
    finally:
        mo.own = False
    return y if isinstance(y, tuple) else (y,)


def off(got, want):
    """How far `got` is from `want`, relative, in the outputs' norm."""
    return ((got.double() - want).norm() / want.norm().clamp(min=1e-30)).item()


# Whole numbers and the scales are exact. A product has four roundings of 2^-24 (relative to values that a bias may make larger
# than the result by a few times), attention in fp32 the sums' of up to 8192 terms; bf16 rounds a result by up to 2^-8, and
# attention its weights too, which a norm over many takes a part of.
LIMIT = {("product", "f32"): 1e-6, ("product", "bf16"): 2.0 ** -8, ("attend", "f32"): 2e-6, ("attend", "bf16"): 4e-3}


def check(case, seed):
    want = mo.exact(case, seed)
    for own in (True, False):
        got = outputs(case, seed, own)
        for g, w in zip(got, want if isinstance(want, tuple) else (want,)):
            if w.numel() == 0:
                continue
            if case["op"] == "quantize":
                assert torch.equal(g.double(), w)
            else:
                assert off(g, w) <= LIMIT[case["op"], case["type"]], own


@pytest.mark.parametrize("name", [c["name"] for c in mo.listed()])
def test_listed(cuda_ok, name):
    check(next(c for c in mo.listed() if c["name"] == name), 3)


@pytest.mark.parametrize("seed", range(24))
def test_drawn(cuda_ok, seed):
    rng = random.Random(seed)
    case = mo.draw(rng)
    while mo.work(case)["flops"] > 2e11:  # (what takes long in 64 bits is left to the listed ones)
        case = mo.draw(rng)
    check(case, seed)
