"""The host side of the operators for sampling, without a GPU: the extension refuses what is not a tensor on the device and counts
its arguments, wrapped tensors and traces stay with the dispatcher, and the C ABI refuses before any launch."""
import pytest
import torch

import q35hip
from q35hip import Q35Error, ops
from test_paged_host import run_with_stubs


def calls():
    h = ops._paged_host()
    kv = torch.zeros(1, 1, 2, 256)
    pages = (torch.zeros(3, 2, 16, 256, dtype=torch.bfloat16),) * 2 + (None, None)
    at = (torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), None)
    rope = (torch.zeros(32, 32), torch.zeros(32, 32), None)
    cuts = (None, 1.0, None, 0, None, 1.0, None, 0.0)
    x, w = torch.zeros(3, 64), torch.zeros(64)
    q, s, W = torch.zeros(3, 64, dtype=torch.int8), torch.zeros(3), torch.zeros(5, 64, dtype=torch.int8)
    return [(h.gated_attn_paged_shared, (kv, None, *pages, *at, *rope, 1e-6, 0.0625, False, 1)),
            (h.sample_tokens, (x, torch.zeros(3), *cuts, False)), (h.filter_logits, (x, *cuts)), (h.quantize_rows_i8, (x,)),
            (h.add_rmsnorm_i8_, (x, None, w, 1e-6)), (h.gemm_i8_, (q, s, W, torch.zeros(5), None, 0, None, 1, None))]


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
    with pytest.raises(TypeError):
        ops._paged_host().bind_sampling(1, 2)


BIND = """
h.bind_sampling(*(ctypes.cast(f, ctypes.c_void_p).value for f in (size, call, size, call, call, call, call)))
logits, w, draws = fake(4, 3, 50), fake(64), fake(4, 3)
rows, W, ws = fake(4, 3, 64), fake(6, 64, dtype=torch.int8), fake(6)
"""


def test_wrapped_tensors_go_through_the_dispatcher():
    out = run_with_stubs(BIND + """
def shapes(t):
    return [tuple(a.shape) for a in (t if isinstance(t, tuple) else (t,))]

print("mapped", shapes(torch.vmap(lambda x: ops.sample_tokens(x, draws[0], top_k=3, want_probs=True))(logits)))
print("mapped", shapes(torch.vmap(lambda u: ops.sample_tokens(logits[0], u))(draws)))
print("mapped", shapes(torch.vmap(lambda x: ops.filter_logits(x, top_p=0.5))(logits)))
print("mapped", shapes(torch.vmap(lambda x: tuple(ops.quantize_rows(x)))(rows)))
print("mapped", shapes(torch.vmap(lambda q: ops.gated_attention_paged_shared(q, None, pages, *at, *rope, 1))(kv)))
print("called", len(done))
""")
    for line in ("mapped [(4, 3), (4, 3, 50)]\nmapped [(4, 3)]\nmapped [(4, 3, 50)]\nmapped [(4, 3, 64), (4, 3)]",
                 "mapped [(3, 1, 1, 512)]", "called 0"):
        assert line in out, out


def test_a_tensor_without_storage_raises():
    out = run_with_stubs(BIND + """
cuts = (None, 1.0, None, 0, None, 1.0, None, 0.0)
for f, arg in [(lambda x: h.sample_tokens(x, draws[0], *cuts, False), logits), (lambda x: h.filter_logits(x, *cuts), logits),
               (lambda x: h.quantize_rows_i8(x), rows), (lambda x: h.add_rmsnorm_i8_(x, None, w, 1e-6), rows),
               (lambda s: h.gemm_i8_(W, s, W, ws, None, 0, None, 1, None), torch.stack([ws] * 2)),
               (lambda q: h.gated_attn_paged_shared(q, None, *pages, *at, None, *rope, None, 1e-6, 0.1, False, 1), kv)]:
    try:
        torch.vmap(lambda t: (f(t), t)[1])(arg)
    except RuntimeError:
        print("raised")
print("called", len(done))
""")
    assert out.count("raised") == 6 and "called 0" in out, out


def test_a_compiled_function_holds_the_ops_whole():
    out = run_with_stubs(BIND + """
seen = []

def backend(gm, inputs):
    seen.extend(str(n.target) for n in gm.graph.nodes if "q35" in str(n.target))
    return gm.forward

def step(q, x, y, u):
    o = ops.gated_attention_paged_shared(q, None, pages, *at, *rope, 1)
    r = ops.add_rmsnorm_i8_(x, y, w)
    a = ops.gemm_i8(ops.quantize_rows(x), W, ws, epilogue="swiglu")
    t = ops.sample_tokens(ops.filter_logits(logits[0], top_k=9), u, top_p=0.9)
    return o, *r, ops.gemm_i8(r, W, ws), a, t

r = torch.compile(step, fullgraph=True, backend=backend)(kv[0], rows[0], rows[1], draws[0])
print([tuple(t.shape) for t in r], *seen)
""")
    assert "[(1, 1, 512), (3, 64), (3,), (3, 6), (3, 3), (3,)]" in out, out
    for name in ("gated_attn_paged_shared", "add_rmsnorm_i8_", "quantize_rows_i8", "gemm_i8_", "filter_logits", "sample_tokens"):
        assert f"q35.{name}" in out, out


def test_the_c_abi_rejects_without_launching():
    L, f, nan = q35hip.lib(), 0x1000, float("nan")
    # rows in 8 bits: no pointer, K not in quads or too long, strides, alignment, other types
    assert L.q35_quantize_rows_i8(None, 64, 0, f, f, 1, 64, None) == 1
    assert L.q35_quantize_rows_i8(f, 60, 0, f, f, 1, 64, None) == 1
    for K, ld, dt, p in ((62, 64, 0, f), (16388, 16388, 0, f), (64, 66, 0, f), (64, 64, 2, f), (64, 64, 0, f + 4), (64, 64, 1, f + 4)):
        assert L.q35_quantize_rows_i8(p, ld, dt, f, f, 2, K, None) == 2
    assert L.q35_add_rmsnorm_i8(f, 64, None, 0, None, f, f, 1, 64, 1e-6, None) == 1
    assert L.q35_add_rmsnorm_i8(f, 64, f, 60, f, f, f, 1, 64, 1e-6, None) == 1
    assert L.q35_add_rmsnorm_i8(f, 64, f + 4, 64, f, f, f, 1, 64, 1e-6, None) == 2

    def gemm(q=f, ldq=64, W=f, y=f, ldy=8, M=4, N=8, K=64, epi=0, pushes=None, npush=0, T=1, cap=None, ldc=0, ldr=0):
        return L.q35_gemm_i8(q, ldq, f, W, f, y, ldy, M, N, K, epi, pushes, npush, T, cap, ldc, ldr, None)
    for bad in (dict(q=None), dict(M=0), dict(ldq=32), dict(ldy=7), dict(epi=3), dict(epi=2, N=7), dict(epi=2, ldy=3), dict(T=0),
                dict(npush=1), dict(pushes=f, npush=65), dict(cap=f, ldc=8, ldr=8), dict(epi=2, cap=f, ldc=3, ldr=4)):
        assert gemm(**bad) == 1, bad
    for bad in (dict(K=32), dict(K=65600, ldq=65600), dict(ldq=72), dict(q=f + 8), dict(W=f + 8), dict(M=1 << 31)):
        assert gemm(**bad) == 2, bad

    size = L.q35_sample_tokens_workspace_bytes
    need = size(2, 1, 1000)
    assert need > 0 and size(2, 1, (1 << 22) + 1) == 0 and size(65536, 1, 5) == 0 and size(300, 300, 5) == 0 and size(0, 1, 5) == 0

    def sample(x=f, u=f, t=1.0, k=0, p=1.0, m=0.0, tok=f, kind=0, out=None, B=2, P=1, V=1000, ws=f, n=need, sb=1000, sp=1000):
        return L.q35_sample_tokens(x, sb, sp, u, 1, None, t, None, k, None, p, None, m, tok, kind, out, B, P, V, ws, n, None)
    for bad in (dict(x=None), dict(u=None), dict(tok=None), dict(t=-1.0), dict(t=nan), dict(p=nan), dict(m=nan), dict(kind=1),
                dict(kind=3, out=f), dict(out=f), dict(P=2), dict(B=0), dict(sb=-1), dict(tok=None, kind=2, out=f, P=2, sp=999)):
        assert sample(**bad) == 1, bad
    assert sample(V=(1 << 22) + 1) == 2
    assert sample(n=need - 1) == 3 and sample(ws=None) == 3 and sample(ws=f + 4) == 3

    size = L.q35_gated_attn_paged_shared_workspace_bytes
    need = size(3, 1, 8, 2, 256, 10, 16, 4)
    assert need > 0 and size(3, 1, 8, 2, 256, 10, 16, 11) == 0 and size(3, 1, 8, 2, 256, 10, 16, -1) == 0
    assert size(3, 1, 8, 2, 256, 10, 16, 0) == L.q35_gated_attn_paged_workspace_bytes(3, 1, 8, 2, 256, 10, 16, 0)

    def attend(shared=4, ws=f, n=need, B=3, T=1, q=f, table=f):
        return L.q35_gated_attn_paged_shared(q, 2048, 2048, 256, None, 0, 0, 0, 0, None, 1e-6, f, f, 64, f, f, None, None, 1, 9, 16,
                                             table, 10, 10, shared, f, None, f, 0, B, T, 8, 2, 256, 0.1, ws, n, None)
    for bad in (dict(shared=-1), dict(shared=11), dict(q=None), dict(table=None)):
        assert attend(**bad) == 1, bad
    assert attend(n=need - 1) == 3 and attend(ws=None) == 3 and attend(ws=f + 8) == 3
    assert attend(B=4, T=1 << 21, n=1 << 50) == 2  # rows of all sequences past 2^24
