"""The layers' rotation tables without a GPU: what a stream capture may ask of them, and which ones a paged layer takes."""
import pytest
import torch

from q35hip import Q35Error, layers


@pytest.fixture(autouse=True)
def empty_cache(monkeypatch):
    monkeypatch.setattr(layers, "_ROPE_CACHE", {})


def test_new_tables_are_refused_inside_a_capture(monkeypatch):
    """Building them waits for a copy, which a capture does not survive: an error of the package's ahead of it."""
    there = layers.rope_tables(64, 64, 1e7, "cpu")
    layers._ROPE_CACHE[(64, 64, 1e7, "cuda:0")] = there
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    assert layers.rope_tables(64, 64, 1e7, torch.device("cuda:0")) is there
    for new in ((128, 64, 1e7), (64, 32, 1e7), (64, 64, 1e4)):
        with pytest.raises(Q35Error, match="capture"):
            layers.rope_tables(*new, torch.device("cuda:0"))


def test_a_paged_layer_takes_tables_that_are_there():
    """Capacities that grow make tables of powers of two, and none is made or dropped for one that fits those there are."""
    for capacity, n in ((0, 1), (100, 128), (128, 128), (90, 128), (129, 256), (100, 128), (5000, 8192), (300, 8192)):
        cos, sin = layers._rope_tables_over(capacity, 64, 1e7, "cpu")
        assert cos.shape == sin.shape == (n, 32)
    assert sorted(k[0] for k in layers._ROPE_CACHE) == [1, 128, 256, 8192]
    long = layers._rope_tables_over(8192, 64, 1e7, "cpu")[0]
    assert torch.equal(long[:128], layers.rope_tables(128, 64, 1e7, "cpu")[0])
    assert layers._rope_tables_over(100, 32, 1e7, "cpu")[0].shape == (128, 16)
