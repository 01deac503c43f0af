"""The inputs of perf/operators.py: a case and a seed give the same ones each time they are made."""
import importlib.util
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


def _cases():
    spec = importlib.util.spec_from_file_location("operator_cases", Path(__file__).resolve().parents[1] / "perf" / "operators.py")
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize("case", [
    # 24 likely ids a row: in a quarter of these rows one of them comes twice
    dict(op="sample", rows=112, vocab=1148, bf16=False, kind="mixed", masked=True),
    dict(op="sample", rows=118, vocab=7126, bf16=True, kind="none", masked=False),
    dict(op="append", n_seq=3, rows=40, ctx=64, heads=8, kv=2, hd=128, page=16, bits=4, f32=False, norm=True, rot=128,
         pairs=False),
    dict(op="attend", n_seq=3, new=4, ctx=200, heads=8, kv=2, hd=128, page=16, bits=16),
], ids=lambda c: f"{c['op']}{c.get('rows', c.get('ctx'))}")
def test_inputs_repeat(case):
    import torch
    m = _cases()
    for seed in range(8):
        a, b = m.prepare(case, seed), m.prepare(case, seed)
        for k, v in a.items():
            if isinstance(v, torch.Tensor):
                same = torch.equal(v.contiguous().view(torch.uint8), b[k].contiguous().view(torch.uint8))
                assert same, (seed, k)
