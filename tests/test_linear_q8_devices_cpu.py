"""What the choice of an 8-bit product's kernel asks of a device, it asks of the device that the weight is on, whichever is the current one."""
import pytest

from arle_b200 import ops


class _Library:
    """Stands for the CUDA library: devices with different numbers of clusters; the current device is 0."""

    clusters = {0: 74, 1: 10}

    def __init__(self):
        self.asked = []

    def arle_gemm_q8_split_clusters(self, parts, device=0):
        self.asked.append((parts, device))
        return self.clusters[device] // parts or 1


@pytest.fixture
def fake(monkeypatch):
    lib = _Library()
    monkeypatch.setattr(ops, "library", lambda: lib)
    monkeypatch.setattr(ops, "_LIB", lib)
    monkeypatch.setattr(ops, "sm_count", lambda device: {0: 148, 1: 20}[device])
    caches = (ops._q8_clusters, ops._q8_route, ops._q8_gate_in_pair)
    for c in caches:
        c.cache_clear()
    yield lib
    for c in caches:
        c.cache_clear()


def test_clusters_are_those_of_the_weight_s_device(fake):
    assert ops._q8_clusters(2, 1) == 5 and ops._q8_clusters(2, 0) == 37
    assert fake.asked == [(2, 1), (2, 0)]


def test_routes_of_two_devices(fake):
    """A route found for one device, its clusters asked for there, and another for the next: neither takes the other's."""
    first, second = (ops._q8_route(200, 4096, 32, d) for d in (1, 0))
    assert {d for _, d in fake.asked} == {0, 1}
    for c in (ops._q8_clusters, ops._q8_route):
        c.cache_clear()
    assert ops._q8_route(200, 4096, 32, 0) == second and ops._q8_route(200, 4096, 32, 1) == first and first != second
