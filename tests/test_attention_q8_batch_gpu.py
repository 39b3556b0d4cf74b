"""Where a batch's tables and the sinks lie, for attention over the 8-bit cache."""
import pytest
import torch

from arle_b200 import ops
from test_attention_q8_gpu import DEV, _case, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("what", ["q_indptr", "kv_lens"])
def test_a_batch_of_another_device_is_refused(what):
    s = _case([(1, 70)], 8, 2, 128, 16)
    setattr(s.batch, what, getattr(s.batch, what).cpu())
    with pytest.raises(ops.KernelError, match="cpu"):
        _run(s)


def test_sinks_of_another_device_are_refused():
    s = _case([(1, 70)], 8, 2, 128, 16)
    for batch in (True, False):
        with pytest.raises(ops.KernelError, match="cpu"):
            _run(s, sink=torch.zeros(8), batch=batch)
        assert _run(s, sink=torch.zeros(8, device=DEV), batch=batch).isfinite().all()
