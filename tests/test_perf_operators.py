"""The plain forms of perf/operators.py against its 64-bit ones, on the host at
small sizes: pages of any size, ragged batches, the rows behind the last sequence."""
import random
import types
from pathlib import Path

import pytest
import torch

SOURCE = Path(__file__).resolve().parents[1] / "perf" / "operators.py"


@pytest.fixture(scope="module")
def ops():
    module = types.ModuleType("operators_on_the_host")
    exec(compile(SOURCE.read_text().replace('"cuda"', '"cpu"'), str(SOURCE), "exec"), module.__dict__)
    return module


def small(ops, seed):
    """A drawn case cut down to what the host computes at once."""
    rng = random.Random(seed)
    case = ops.draw(rng)
    if case["kind"] == "sample":
        case.update(rows=min(case["rows"], 5), vocab=min(case["vocab"], 700))
        return case
    case.update(sequences=min(case["sequences"], 3), heads=case["kv_heads"] * min(2, case["heads"] // case["kv_heads"]),
                new=min(case["new"], 9), length=min(case["length"], rng.randint(9, 40)))
    case["page_size"] = rng.choice([1, 1, 2, 3, 5, 16])
    if case["kind"] == "attention" and case["window"]:
        case["window"] = min(case["window"], rng.randint(1, 20))
    return case


def tensors(out):
    return list(out.values()) if isinstance(out, dict) else [out]


@pytest.mark.parametrize("seed", range(60))
def test_plain_forms_agree_with_64_bits(ops, seed):
    """Each output within half a step of its type and, for what is summed in 32 bits
    before that, 2^-12 of the largest: a dot of 256 products errs by some 2^-20 of
    its terms' sum, which lies below 2^4 here, a weight by twice that, 2^-15."""
    case = small(ops, seed)
    got = tensors(ops.run(ops.prepare(case, seed)))
    for g, want in zip(got, tensors(ops.exact(case, seed))):
        if want is None:
            continue
        step = torch.finfo(g.dtype).eps / 2
        want = want.double()
        assert ((g.double() - want).abs() <= step * want.abs() + 2.0 ** -12 * want.abs().max()).all(), case


@pytest.mark.parametrize("page_size", [1, 2, 3, 4, 10, 16])
@pytest.mark.parametrize("length", [10, 12])
def test_rotary_rows_behind_the_last_sequence_have_no_page(ops, page_size, length):
    """Sequences that fill their pages, with the two rows behind the last one: these
    stay as they are, and nothing is looked up for them."""
    case = ops._rope("", sequences=3, new=4, length=length, heads=2, kv_heads=1, head_dim=16, dims=16, page_size=page_size)
    state = ops.prepare(case, 5)
    before = state["q_out"].clone()
    got = ops.run(state)
    assert torch.equal(got["q"][-2:], before[-2:]) and (got["q"][:-2] != 0).any()
    for g, want in zip(got.values(), ops.exact(case, 5).values()):
        assert ((g.double() - want).abs() <= torch.finfo(g.dtype).eps * want.abs() + 2.0 ** -20).all()
