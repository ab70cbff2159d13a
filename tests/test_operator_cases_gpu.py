"""perf/operators.py on the GPU: for every listed case, made smaller, and for
drawn ones, the library's calls and the plain form both give what the file's
64-bit form does.

Tolerances: a sum of n terms in fp32 is off by at most n * 2^-24 times the sum
of the terms' magnitudes (one more step for the products), and the result's
rounding adds half a step of its type.  Whole numbers and moved rows are equal."""
import importlib.util
import os
import random

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "perf",
                    "operators.py")
HALF = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
TINY = {torch.float32: 2.0**-149, torch.float16: 2.0**-24, torch.bfloat16: 2.0**-133}


@pytest.fixture
def ops():
    spec = importlib.util.spec_from_file_location("operator_cases", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def smaller(case):
    """The same form of a case with fewer tokens or positions."""
    c = dict(case)
    if "T" in c:
        c["T"] = min(c["T"], 2501 if c["op"] != "sort" else 40_001)
    if "S" in c and c["S"] > 4104:
        f = 4104 / c["S"]
        c["S"] = 4104
        for k in ("budget", "recent"):
            if k in c:
                c[k] = max(1, int(c[k] * f))
    c["B"] = min(c.get("B", 1), 4)
    return c


def cases():
    spec = importlib.util.spec_from_file_location("operator_cases", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    out = [(c["name"], smaller(c)) for c in module.listed()]
    rng = random.Random(4)
    while len(out) < 32:
        c = module.draw(rng)
        if module.work(c)["bytes"] < 1.5e8:
            out.append((f"draw{len(out)}-{c['op']}", c))
    return out


CASES = cases()


def magnitudes(ops, case, seed):
    """The exact outputs for the inputs' magnitudes: the sums of the terms'."""
    s = ops.prepare(case, seed)
    for name in ("weights", "x", "expert_out", "grad_y", "grad_rows", "scores"):
        if name in s:
            s[name] = s[name].abs()
    return {"experts": ops._exact_experts, "add": ops._exact_add}[
        "add" if case["op"] == "add" else "experts"](case, s)


def terms_of(case, name):
    if case["op"] == "add":
        return case["Hq"] // case["Hkv"] * case["Q"] + 1
    return {"y": case["K"], "grad_out": 0, "grad_x": case["K"], "grad_weights": case["H"]}[name]


SUMS = ("y", "grad_out", "grad_x", "grad_weights", "totals")


@pytest.mark.parametrize("name,case", CASES, ids=[n for n, _ in CASES])
@pytest.mark.parametrize("own", [True, False])
def test_a_case_gives_its_exact_outputs(ops, name, case, own):
    ops.own = own
    got, want = ops.run(ops.prepare(case, 7)), ops.exact(case, 7)
    if case["op"] == "add":
        got, want = {"totals": got}, {"totals": want}
    mags = None
    assert got.keys() == want.keys()
    for k, w in want.items():
        g = got[k]
        if isinstance(w, np.ndarray):
            w = torch.from_numpy(w).cuda()
        assert g.shape == w.shape
        if k not in SUMS:
            assert torch.equal(g.to(w.dtype), w), k
            continue
        if mags is None:
            mags = magnitudes(ops, case, 7)
            mags = {"totals": mags} if case["op"] == "add" else mags
        tol = (terms_of(case, k) + 1) * 2.0**-24 * mags[k]
        tol = tol + HALF[g.dtype] * (w.abs() + tol) + TINY[g.dtype]
        assert torch.isfinite(g).all()
        assert ((g.double() - w).abs() <= tol).all(), k
