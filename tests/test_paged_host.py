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


# The extension bound to entry points that do nothing, for tensors on a device that is not there. In a process of its own: a
# fault in it ends that process, and the binding is for good.
STUBS = """
import ctypes
import sys
sys.path.insert(0, {root!r})
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from q35hip import Q35Error, _lib, ops

h = ops._paged_host()
done = []
call = ctypes.CFUNCTYPE(ctypes.c_int)(lambda: done.append(1) or 0)
size = ctypes.CFUNCTYPE(ctypes.c_size_t)(lambda: 256)
h.bind(Q35Error, _lib.check, lambda d: 0, *(ctypes.cast(f, ctypes.c_void_p).value for f in (call, call, size, call, size, call)))


def fake(*size, dtype=torch.float32):
    with FakeTensorMode(allow_non_fake_inputs=True):
        return torch.zeros(*size, dtype=dtype, device="cuda:0")


kv, x, u = fake(3, 1, 1, 2, 256), fake(3, 1, 2, 5), fake(3, 1, 2)  # three of each, to be mapped over
pages = (*(fake(3, 2, 16, 256, dtype=torch.bfloat16) for _ in range(2)), None, None)
at = (fake(1, 2, dtype=torch.int32), fake(1, dtype=torch.int32))
rope = (fake(32, 32), fake(32, 32))
ids = fake(1, 1, dtype=torch.int32)
"""


def run_with_stubs(body):
    import os
    import subprocess
    import sys
    import textwrap
    from q35hip import build
    r = subprocess.run([sys.executable, "-c", STUBS.format(root=build.ROOT) + textwrap.dedent(body)], capture_output=True,
                       text=True, timeout=300, env=dict(os.environ, PYTHONFAULTHANDLER="1"))
    assert r.returncode == 0, r.stdout + r.stderr[-3000:]
    return r.stdout


def test_a_tensor_without_storage_raises():
    """A wrapper of functorch's has no address to give: an exception out of the extension, with the interpreter lock held."""
    out = run_with_stubs("""
        calls = [(lambda k: h.paged_kv_append(k, k, *pages, *at, None, *rope, None, 1e-6), kv),
                 (lambda p: h.paged_kv_rows(p, p, None, None, *at, None, 4), torch.stack([pages[0]] * 3)),
                 (lambda q: h.gated_attn_paged(q, None, *pages, *at, None, *rope, None, 1e-6, 0.1, 0, False), kv),
                 (lambda u: h.verify_drafts(x[0], ids, None, u, None, None, 1.0), u)]
        for f, arg in calls:
            try:
                torch.vmap(lambda t: (f(t), t)[1])(arg)
            except RuntimeError as e:
                print("raised", type(e).__name__, "storage" in str(e))
        print("called", len(done))
        """)
    assert out.count("raised") == 4 and "called 0" in out, out


def test_wrapped_tensors_go_through_the_dispatcher():
    """vmap, functionalization and a tensor that is negated when read, in any argument: none reaches the extension."""
    out = run_with_stubs("""
        logits = torch.stack([x[0]] * 3)
        n, tok = torch.vmap(lambda l: ops.verify_drafts(l, ids, u[0]))(logits)
        print("mapped", tuple(n.shape), tuple(tok.shape))
        n, tok = torch.vmap(lambda w: ops.verify_drafts(x[0], ids, w))(u)  # (the first argument is not wrapped)
        print("mapped", tuple(n.shape), tuple(tok.shape))
        o = torch.vmap(lambda q: ops.gated_attention_paged(q, None, pages, *at, *rope))(kv)
        print("mapped", tuple(o.shape))
        o, _ = torch.vmap(lambda p: ops.paged_kv_rows((p, p), *at, 4))(torch.stack([pages[0]] * 3))
        print("mapped", tuple(o.shape))
        o = ops.gated_attention_paged(torch._to_functional_tensor(kv[0]), None, pages, *at, *rope)
        print("functional", tuple(o.shape))
        with torch.enable_grad():
            print("direct", h.direct(kv[0]), h.direct(torch._to_functional_tensor(kv[0])), h.direct(1.0, None),
                  h.direct(torch.zeros(2)))
        print("called", len(done))
        """)
    for line in ("mapped (3, 1) (3, 1, 2)\nmapped (3, 1) (3, 1, 2)\nmapped (3, 1, 1, 512)\nmapped (3, 1, 2, 4, 256)",
                 "functional (1, 1, 512)", "direct False False True False", "called 0"):
        assert line in out, out


def test_a_compiled_function_holds_the_ops_whole():
    """torch.compile without a break in the graph, for all four."""
    out = run_with_stubs("""
        seen = []

        def backend(gm, inputs):
            seen.extend(str(n.target) for n in gm.graph.nodes if "q35" in str(n.target))
            return gm.forward

        def step(k, q, u):
            ops.paged_kv_append_(k, k, pages, *at, *rope)
            a, _ = ops.paged_kv_rows(pages, *at, 4)
            o = ops.gated_attention_paged(q, None, pages, *at, *rope)
            return a, o, *ops.verify_drafts(x[0], ids, u, temperature=0.5)

        r = torch.compile(step, fullgraph=True, backend=backend)(kv[0], kv[0], u[0])
        print([tuple(t.shape) for t in r], len(seen), *seen)
        """)
    assert "[(1, 2, 4, 256), (1, 1, 512), (1,), (1, 2)] 4" in out, out
    for name in ("paged_kv_append_", "paged_kv_rows", "gated_attn_paged", "verify_drafts"):
        assert f"q35.{name}" in out, out


def test_a_trace_records_the_ops(monkeypatch):
    """torch.jit.trace and a dispatch mode, over tensors that pass for device ones: nothing but torch.ops is called."""
    from torch.utils._python_dispatch import TorchDispatchMode
    host, called = ops._paged_host(), []

    class Host:  # (asks what is asked of the thread, not of the tensors)
        def __getattr__(self, name):
            return lambda *args: (called.append(name), (args[0], args[1]))[1] if host.direct() else NotImplemented
    monkeypatch.setattr(ops, "_HOST", Host())

    def meta(*size, dtype=torch.float32):
        return torch.zeros(*size, dtype=dtype, device="meta")
    args = (meta(1, 1, 2, 256), meta(3, 2, 16, 256, dtype=torch.bfloat16), meta(1, 2, dtype=torch.int32),
            meta(1, dtype=torch.int32), meta(32, 32), meta(1, 2, 5), meta(1, 1, dtype=torch.int32), meta(1, 2))

    def step(kv, page, table, pos, rope, x, ids, u):
        ops.paged_kv_append_(kv, kv, (page, page), table, pos, rope, rope)
        o = ops.gated_attention_paged(kv, None, (page, page), table, pos, rope, rope)
        o = o[0] if isinstance(o, tuple) else o
        return o, *ops.paged_kv_rows((page, page), table, pos, 4), *ops.verify_drafts(x, ids, u)
    with monkeypatch.context() as m:
        m.setattr(torch.Tensor, "is_cuda", property(lambda t: True))
        step(*args)
        assert len(called) == 4
        called.clear()
        graph = torch.jit.trace(step, args, check_trace=False).inlined_graph
        recorded = [n.kind() for n in graph.nodes()]
        seen = []

        class Record(TorchDispatchMode):
            def __torch_dispatch__(self, func, types, args=(), kwargs=None):
                seen.append(str(func))
                return func(*args, **(kwargs or {}))
        with Record():
            step(*args)
    assert not called
    for name in ("paged_kv_append_", "paged_kv_rows", "gated_attn_paged", "verify_drafts"):
        assert f"q35::{name}" in recorded and f"q35.{name}.default" in seen, (name, recorded, seen)
