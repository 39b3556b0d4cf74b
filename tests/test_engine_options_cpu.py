"""Options by position keep their meaning: a new one goes behind those that were there."""
from dataclasses import fields

from arle_b200.engine.engine import EngineOptions

EARLIER = ["dtype", "device", "page_size", "num_pages", "mem_fraction_static", "num_slots", "max_seq_len", "max_num_batched_tokens", "chunked_prefill_size", "max_prefill_tokens",
           "prefill_max_requests", "scheduler_mixed_policy", "max_tokens", "seed", "cuda_graph", "kernel_set", "cache_dtype", "device_tables"]


def test_options_by_position():
    names = [f.name for f in fields(EngineOptions)]
    assert names[: len(EARLIER)] == EARLIER and "weight_dtype" in names[len(EARLIER):]
    values = [f.default for f in fields(EngineOptions)][: len(EARLIER) - 2] + ["float8_e4m3", True]
    o = EngineOptions(*values)
    assert (o.cache_dtype, o.device_tables, o.weight_dtype) == ("float8_e4m3", True, "auto")
