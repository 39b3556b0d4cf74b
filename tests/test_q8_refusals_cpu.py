"""What the operators of the 8-bit cache and the step's tables refuse, before anything is launched."""
import pytest
import torch

from arle_b200 import ops

BF, F8, F32, I32 = torch.bfloat16, torch.float8_e4m3fn, torch.float32, torch.int32


def _cache(pages=3, nkv=2, ps=16, hd=64, vd=64):
    return dict(k_cache=torch.zeros(pages, nkv, ps, hd, dtype=F8), v_cache=torch.zeros(pages, nkv, ps, vd, dtype=F8), k_scale=torch.zeros(pages, nkv),
                v_scale=torch.zeros(pages, nkv))


def _store(**changed):
    a = dict(k=torch.zeros(4, 128, dtype=BF), v=torch.zeros(4, 128, dtype=BF), slot_mapping=torch.zeros(4, dtype=I32), **_cache(), nkv=2, hd=64, page_size=16)
    a.update(changed)
    ops.store_q8(**a)


def _attend(**changed):
    a = dict(q=torch.zeros(4, 256, dtype=BF), out=torch.zeros(4, 256, dtype=BF), **_cache(), positions=torch.zeros(4, dtype=I32), row_of_token=torch.zeros(4, dtype=I32),
             block_table=torch.zeros(1, 1, dtype=I32), nq=4, nkv=2, hd=64, page_size=16, scale=0.1, window=None)
    a.update(changed)
    ops.paged_attention_q8(**a)


CACHES = [dict(k_cache=torch.zeros(3, 2, 16, 64, dtype=torch.uint8)), dict(v_cache=torch.zeros(3, 2, 16, 64, dtype=BF)), dict(k_cache=torch.zeros(3, 2, 8, 64, dtype=F8)),
          dict(v_cache=torch.zeros(4, 2, 16, 64, dtype=F8)), dict(k_cache=torch.zeros(3, 2, 64, 16, dtype=F8).transpose(2, 3)), dict(k_scale=torch.zeros(3, 2, dtype=BF)),
          dict(v_scale=torch.zeros(2, 3).t()), dict(k_scale=torch.zeros(2, 2))]


@pytest.mark.parametrize("changed", CACHES + [dict(k=torch.zeros(4, 64, dtype=BF)), dict(v=torch.zeros(4, 128)), dict(k=torch.zeros(3, 128, dtype=BF)),
                                              dict(k=torch.zeros(128, 4, dtype=BF).t()), dict(slot_mapping=torch.zeros(4, dtype=torch.int64)),
                                              dict(slot_mapping=torch.zeros(8, dtype=I32)[::2]), dict(vd=32), dict(page_size=8), dict(nkv=1)])
def test_store(changed):
    with pytest.raises(ops.KernelError):
        _store(**changed)


@pytest.mark.parametrize("changed", CACHES + [dict(q=torch.zeros(4, 128, dtype=BF)), dict(q=torch.zeros(256, 4, dtype=BF).t()), dict(out=torch.zeros(4, 256)),
                                              dict(out=torch.zeros(4, 512, dtype=BF)[:, :256]), dict(positions=torch.zeros(4)), dict(row_of_token=torch.zeros(4, dtype=torch.int64)),
                                              dict(block_table=torch.zeros(1, 1, dtype=torch.int64)), dict(block_table=torch.zeros(2, 2, dtype=I32).t()), dict(nq=3), dict(vd=32),
                                              dict(sink=torch.zeros(3)), dict(sink=torch.zeros(4, dtype=BF))])
def test_attention(changed):
    with pytest.raises(ops.KernelError):
        _attend(**changed)


def test_tensors_of_the_cpu():
    for call in (_store, _attend):
        with pytest.raises(ops.KernelError, match="CUDA"):
            call()


def _tables(R=2, T=5, width=3, **changed):
    z = lambda *n: torch.zeros(*n, dtype=I32)      # noqa: E731
    a = dict(slots=z(R), starts=z(R), q_lens=z(R), new_pages=z(1), page_table=z(4, 3), num_pages=4, page_size=16, q_indptr=z(R + 1), kv_lens=z(R), positions=z(T),
             row_of_token=z(T), slot_of_token=z(T), slot_mapping=z(T), block_table=z(R, width), status=z(1))
    a.update(changed)
    ops.step_tables(**a)


@pytest.mark.parametrize("name,bad", [("slots", torch.zeros(2)), ("starts", torch.zeros(3, dtype=I32)), ("q_lens", torch.zeros(2, dtype=torch.int64)),
                                      ("new_pages", torch.zeros(4, dtype=I32)[::2]), ("page_table", torch.zeros(12, dtype=I32)), ("page_table", torch.zeros(3, 4, dtype=I32).t()),
                                      ("q_indptr", torch.zeros(2, dtype=I32)), ("kv_lens", torch.zeros(3, dtype=I32)), ("row_of_token", torch.zeros(4, dtype=I32)),
                                      ("slot_of_token", torch.zeros(6, dtype=I32)), ("slot_mapping", torch.zeros(4, dtype=I32)), ("block_table", torch.zeros(3, 3, dtype=I32)),
                                      ("block_table", torch.zeros(2, dtype=I32)), ("status", torch.zeros(2, dtype=I32))])
def test_tables(name, bad):
    with pytest.raises(ops.KernelError):
        _tables(**{name: bad})


def test_tables_of_the_cpu():
    with pytest.raises(ops.KernelError, match="CUDA"):
        _tables()
