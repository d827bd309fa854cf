"""The timed operators' plain form and the library's calls side by side, at sizes where a sequence ends at or next to the end of its last page and
rows of no sequence lie behind it."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def operators():
    spec = importlib.util.spec_from_file_location("timed_operators", os.path.join(ROOT, "perf", "operators.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("op,f32", [("append", False), ("append", True), ("read", False), ("read", True), ("attention", False)])
@pytest.mark.parametrize("longest", [32, 30, 33])
def test_rows_behind_a_full_last_page(op, f32, longest, monkeypatch):
    monkeypatch.chdir(ROOT)
    timed = operators()
    case = dict(op=op, sequences=2, kv_heads=2, head_dim=64, group=32, page=16, longest=longest, new=9, ragged=False, behind=5)
    case.update(dict(heads=4, window=0) if op == "attention" else dict(f32=f32))
    found = []
    for timed.own in (False, True):
        print(op, longest, f32, timed.own, flush=True)
        found.append({k: v.clone() for k, v in timed.run(timed.prepare(case, 3)).items()})
        torch.cuda.synchronize()
    for k, plain in found[0].items():
        assert not plain[:, -5:].any() and not found[1][k][:, -5:].any()
        if op == "attention":  # probabilities and outputs rounded to halfs, of values below 6 or so
            assert (plain.double() - found[1][k].double()).abs().max() <= 6 * 2.0**-11 + 2.0**-11 * plain.double().abs().max()
        else:
            assert torch.equal(plain, found[1][k])
