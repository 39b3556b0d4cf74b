"""What attention over the 8-bit cache asks of its workspace and launches, in which order, with the library's place taken by a list."""
import weakref
from types import SimpleNamespace

import pytest
import torch

from arle_b200 import ops
from arle_b200.engine.batch import Workspace

BF, F8, I32 = torch.bfloat16, torch.float8_e4m3fn, torch.int32


class Recorded(Workspace):
    """A workspace that notes which buffers were made (a zeroed one is a launch) beside the launches."""

    def __init__(self, log):
        super().__init__("cpu")
        self.log = log

    def _noted(self, made, name, shape, dtype):
        before = self.generation
        out = made(name, shape, dtype)
        if self.generation != before:
            self.log.append("made " + name)
        return out

    def get(self, name, shape, dtype):
        return self._noted(super().get, name, shape, dtype)

    def get_zeroed(self, name, shape, dtype):
        return self._noted(super().get_zeroed, name, shape, dtype)


@pytest.fixture
def log(monkeypatch):
    events = []

    class Library:
        def __getattr__(self, name):
            def launch(*args):
                events.append(name)
                return 0
            return launch

    monkeypatch.setattr(ops, "library", lambda: Library())
    monkeypatch.setattr(ops, "_placed", lambda what, tensors: (-1, map(torch.Tensor.data_ptr, tensors)))
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: 0, raising=False)
    monkeypatch.setattr(ops, "_ptr", lambda t, name="tensor": None if t is None else t.data_ptr())
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(ops, "_SM_COUNT", {None: 148, -1: 148})
    monkeypatch.setattr(ops, "error_flag", lambda device: torch.zeros(1, dtype=I32))
    return events


def attend(ws, rows, nq=8, nkv=2, hd=128, ps=16, dtype=BF, change=None):
    """One call; rows: (queries, keys).  ``change``: of the batch and the call's tables."""
    z = lambda *n: torch.zeros(*n, dtype=I32)      # noqa: E731
    lens, kvs = [n for n, _ in rows], [kv for _, kv in rows]
    T, R, width = sum(lens), len(rows), -(-max(kvs) // ps)
    batch = SimpleNamespace(q_indptr=z(R + 1), kv_lens=z(R), q_lens=lens, kv_lens_host=kvs, num_rows=R, max_q_len=max(lens), max_kv_len=max(kvs),
                            num_single=sum(n == 1 for n in lens), ws=ws, memo={})
    cache = [torch.zeros(4, nkv, ps, hd, dtype=F8) for _ in range(2)] + [torch.zeros(4, nkv) for _ in range(2)]
    q = torch.zeros(T, nq * hd, dtype=dtype)
    tables = dict(positions=z(T), row_of_token=z(T), block_table=z(R, width))
    if change is not None:
        change(batch, tables)
    ops.paged_attention_q8(q, torch.empty_like(q), *cache, *tables.values(), nq, nkv, hd, ps, 0.1, None, batch=batch)


@pytest.mark.parametrize("hd", [64, 128])
def test_nothing_comes_between_the_prompt_kernel_and_the_decoded_tokens_beside_it(log, hd):
    """The decoded tokens' kernel starts beside the prompt kernel and waits for its end only when it is done itself, so counters that are made for it are
    zeroed in front of the prompt kernel: at the first mixed step, and where a later one needs more of them."""
    ws = Recorded(log)
    for decoded, grows in ((2, True), (5, True), (5, False), (40, True)):
        del log[:]
        attend(ws, [(1, 700)] * decoded + [(600, 3000)], hd=hd)
        prompt = max(i for i, e in enumerate(log) if e.startswith("arle_paged_attention_prefill"))
        assert log[prompt + 1] == "arle_attention_q8_decode", log
        assert ("made attn_q8_counters" in log[:prompt]) == grows


DECODED, SHORT, LONG = [(1, 70), (1, 300)], [(3, 70), (1, 300)], [(200, 3000), (1, 300)]
I = lambda n, step=1: torch.zeros(n * step, dtype=I32)[::step]      # noqa: E731


def _set(what, value):
    def change(batch, tables):
        if what in tables:
            tables[what] = value
        else:
            setattr(batch, what, value)
    return change


@pytest.mark.parametrize("rows,dtype,what,value", [
    (DECODED, BF, "q_indptr", I(2)), (DECODED, BF, "q_indptr", I(3, 2)), (DECODED, BF, "kv_lens", I(1)), (DECODED, BF, "kv_lens", I(2, 2)),
    (DECODED, BF, "block_table", torch.zeros(1, 19, dtype=I32)), (SHORT, BF, "positions", I(3)), (SHORT, BF, "positions", I(4, 2)), (SHORT, BF, "row_of_token", I(3)),
    (SHORT, BF, "row_of_token", I(4, 3)), (LONG, BF, "q_lens", [200]), (LONG, BF, "kv_lens_host", [3000]), (LONG, BF, "block_table", torch.zeros(1, 188, dtype=I32)),
    (DECODED, torch.float32, "positions", I(1)), (DECODED, torch.float32, "row_of_token", I(2, 2))])
def test_tables_that_are_too_short_or_not_contiguous_are_refused(log, rows, dtype, what, value):
    """Whatever a kernel would read behind the end of, or past the strides of: nothing is launched."""
    ws = Recorded(log)
    attend(ws, rows, dtype=dtype)
    del log[:]
    with pytest.raises(ops.KernelError, match="paged_attention_q8"):
        attend(ws, rows, dtype=dtype, change=_set(what, value))
    assert not log


def test_longer_tables_are_taken(log):
    for what, value in (("q_indptr", I(9)), ("kv_lens", I(5)), ("positions", I(9)), ("row_of_token", I(9)), ("block_table", torch.zeros(5, 19, dtype=I32))):
        attend(Recorded(log), SHORT, change=_set(what, value))


def test_no_kv_heads(log):
    with pytest.raises(ops.KernelError, match="heads"):
        attend(Recorded(log), DECODED, nkv=0)


def test_a_long_prompt_in_portions_makes_few_buffers(log):
    """Every portion sees more keys than the one in front of it; its buffers grow by powers of two."""
    ws = Recorded(log)
    for portion in range(1, 65):
        attend(ws, [(512, 512 * portion)])
    assert max(log.count(e) for e in log if e.startswith("made")) <= 8        # 8 to 512 pages of 64 tokens, with or without their tables


@pytest.mark.parametrize("limit", [1 << 20, 3 << 20, 1 << 30])
@pytest.mark.parametrize("nkv", [2, 3])
def test_what_the_engine_leaves_room_for_is_enough(log, monkeypatch, limit, nkv):
    """Steps of all forms, rows that see more than goes at a time among them, against the bytes that are set aside."""
    monkeypatch.setattr(ops, "Q8_EXPAND_BYTES", limit)
    ws = Recorded(log)
    for rows in ([(300, 700)], [(300, 2100), (1, 900), (200, 200)], [(1, 900)] * 30 + [(700, 1200)] * 2, [(64, 9000), (4000, 4000)], [(2, 8000), (1, 1)], [(600, 9000)] * 3):
        attend(ws, rows, nq=4 * nkv, nkv=nkv)
        big = sum(b.numel() * b.element_size() for (name, _), b in ws._bufs.items() if name not in ("attn_q8_table", "attn_q8_counters"))
        assert big <= ops.q8_scratch_bytes(-(-9000 // 64) * 64 * 2 * 2 * nkv * 128)


@pytest.mark.parametrize("zeroed", [False, True])
def test_a_workspace_lets_go_of_a_buffer_before_it_makes_a_larger_one(monkeypatch, zeroed):
    ws, name = Workspace("cpu"), "zeros" if zeroed else "empty"
    get, make = ws.get_zeroed if zeroed else ws.get, getattr(torch, name)
    first = weakref.ref(get("a", (3, 8), torch.float32))
    ws.cut("a", first(), 0, 4)
    alive = []
    monkeypatch.setattr(torch, name, lambda *a, **k: (alive.append(first() is not None), make(*a, **k))[1])
    assert get("a", (9, 8), torch.float32).shape == (9, 8)
    assert alive == [False]
