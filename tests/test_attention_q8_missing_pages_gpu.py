"""A page of -1 among the keys that a query sees counts as keys and values of zeros in every kernel of the attention over the 8-bit cache."""
import pytest
import torch

from arle_b200 import ops
from test_attention_q8_gpu import BF, DEV, _case, _near, _run, _want

pytestmark = pytest.mark.gpu


def _without_page_0(rows, ps, hd, dtype):
    """A case whose page 0, which some row holds, is gone: NaN in the cache, -1 in the table.  And what the definition makes of it: a page of zeros."""
    s = next(x for x in (_case(rows, 8, 2, hd, ps, dtype=dtype, seed=seed) for seed in range(20)) if (x.table == 0).any())
    gone = s.table == 0
    zeros = s.k.shape[0]
    s.k, s.v = (torch.cat([c.view(torch.uint8), torch.zeros_like(c[:1]).view(torch.uint8)]).view(c.dtype) for c in (s.k, s.v))
    s.ks, s.vs = (torch.cat([x, torch.ones_like(x[:1])]) for x in (s.ks, s.vs))
    for c in (s.k, s.v):
        c.view(torch.uint8)[0] = 0x7f
    for x in (s.ks, s.vs):
        x[0] = float("nan")
    s.table = torch.where(gone, zeros, s.table)
    want = _want(s)
    s.table = torch.where(gone, -1, s.table)
    s.bt = s.table.to(DEV)
    return s, want


@pytest.mark.parametrize("ps", [16, 12, 64])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("form", ["decoded", "by tokens", "expanded", "general", "float32"])
def test_a_page_that_is_not_there(form, ps, hd, monkeypatch):
    monkeypatch.setattr(ops, "_by_tokens_q8", lambda *a: form == "by tokens")
    rows = [(1, 130)] * 4 if form == "decoded" else [(70, 130)] * 4
    s, want = _without_page_0(rows, ps, hd, torch.float32 if form == "float32" else BF)
    _near(_run(s, batch=form != "general"), want, hd, {"expanded": 2.0 ** -8, "general": 0.0, "float32": 0.0}.get(form, 2.0 ** -11), 130)
    ops.check_errors(DEV)


@pytest.mark.parametrize("hd,vd", [(33, 33), (128, 128)])
def test_an_empty_steps_queries_get_zeros(hd, vd):
    """The general kernel on what step_tables leaves of a step that is not in order; pages carry NaN."""
    s = _case([(3, 50)], 2, 2, hd, 16, dtype=torch.float32, vd=vd)
    for c in (s.k, s.v):
        c.view(torch.uint8).fill_(0x7f)
    for x in (s.positions, s.row_of):
        x.zero_()
    s.bt.fill_(-1)
    assert not _run(s, batch=False).any()
