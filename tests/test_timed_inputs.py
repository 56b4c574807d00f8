"""perf/more_operators.py: a case's inputs come from its seed alone, not from the order in which a GPU's threads happen to
write."""
import importlib.util
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parents[1]


def load():
    spec = importlib.util.spec_from_file_location("timed_more_operators", ROOT / "perf" / "more_operators.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.fixture
def timed(monkeypatch):
    module = load()
    monkeypatch.setattr(module, "DEV", "cpu")
    return module


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
def test_logits_do_not_depend_on_the_order_of_writes(timed, monkeypatch, masked, dtype):
    """Rows in which a likely token is drawn twice, all scattered writes in order and in the opposite one."""
    case = dict(op="score", dtype=dtype, rows=77, vocab=1000, top=5, masked=masked)
    first = [timed.prepare(case, seed) for seed in range(3)]

    def backwards(real):
        return lambda x, dim, index, src, *args, **kw: real(x, dim, index.flip(dim), src.flip(dim), *args, **kw)

    for name in ("scatter_", "scatter_add_", "scatter_reduce_"):
        monkeypatch.setattr(torch.Tensor, name, backwards(getattr(torch.Tensor, name)))
    for seed, st in enumerate(first):
        other = timed.prepare(case, seed)
        assert torch.equal(st["logits"], other["logits"]) and torch.equal(st["tokens"], other["tokens"]), seed


def test_seeds_differ(timed):
    case = dict(op="score", dtype="float32", rows=7, vocab=1000, top=5, masked=True)
    a, b = (timed.prepare(case, seed)["logits"] for seed in (1, 2))
    assert not torch.equal(a, b) and torch.isinf(a).sum() > 6000


@pytest.mark.gpu
def test_a_seed_gives_the_same_logits_on_a_gpu():
    """50 seeds of the masked case, of which about 18 have a row with a token drawn twice."""
    timed = load()
    case = next(c for c in timed.listed() if c["name"] == "score_masked")
    for seed in range(50):
        a, b = (timed.prepare(case, seed) for _ in range(2))
        assert torch.equal(a["logits"], b["logits"]) and torch.equal(a["tokens"], b["tokens"]), seed
