"""The host extension of the paged-cache ops without a GPU: it loads, counts its arguments and refuses what is not a tensor on
the device with the package's error."""
import pytest
import torch

from q35hip import Q35Error, ops


def calls():
    h = ops._paged_host()
    kv = torch.zeros(1, 1, 2, 256)
    pages = (torch.zeros(3, 2, 16, 256, dtype=torch.bfloat16),) * 2 + (None, None)
    at = (torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), None)
    rope = (torch.zeros(32, 32), torch.zeros(32, 32), None)
    ids = torch.zeros(1, 0, dtype=torch.int32)
    return [(h.paged_kv_append, (kv, kv, *pages, *at, *rope, 1e-6)), (h.paged_kv_rows, (*pages, *at, 4)),
            (h.gated_attn_paged, (kv, None, *pages, *at, *rope, 1e-6, 0.0625, 0, False)),
            (h.verify_drafts, (torch.zeros(1, 1, 5), ids, None, torch.zeros(1, 1), None, None, 1.0))]


def test_tensors_off_the_device_are_refused():
    for f, args in calls():
        with pytest.raises(Q35Error, match="HIP device tensors"):
            f(*args)
        with pytest.raises(Q35Error, match="HIP device tensors"):
            f(*(a.to("meta") if torch.is_tensor(a) else a for a in args))


def test_arguments_are_counted_and_typed():
    for f, args in calls():
        for bad in (args[:-1], args + (None,), ()):
            with pytest.raises(Q35Error, match="number of arguments"):
                f(*bad)
        for what in (None, 3.0, [1], "x"):
            with pytest.raises(Q35Error, match="must be tensors"):
                f(what, *args[1:])
    f, args = calls()[3]
    with pytest.raises(TypeError):
        f(*args[:-1], "warm")


def test_bind_takes_nine_arguments():
    with pytest.raises(TypeError):
        ops._paged_host().bind(Q35Error)
