"""The benchmark's option for weights in 8 bits stays out of the contract's run, which is of 16 bits."""
import sys

import pytest

import bench


@pytest.mark.parametrize("more", [[], ["--only", "gemm"], ["--design", "kolodra"]])
def test_weights_in_8_bits_go_with_decode_or_prefill_alone(more, monkeypatch, capsys):
    monkeypatch.setattr(sys, "argv", ["bench.py", "--weight-dtype", "float8_e4m3", *more])
    assert bench.main() == 2 and "--weight-dtype" in capsys.readouterr().out
