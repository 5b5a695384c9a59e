"""Group norm and differential attention without a GPU: the restatements'
gradients against differences, and what the calls refuse."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import block_ref as B


def _central(f, x, step=1e-5):
    g = np.zeros_like(x)
    it = np.nditer(x, flags=["multi_index"])
    for _ in it:
        i = it.multi_index
        keep = x[i]
        x[i] = keep + step
        a = f()
        x[i] = keep - step
        b = f()
        x[i] = keep
        g[i] = (a - b) / (2 * step)
    return g


@pytest.mark.parametrize("silu", [False, True])
def test_group_norm_gradient_against_differences(silu):
    rng = np.random.default_rng(0)
    cu = [0, 3, 3, 4, 9]
    x, dy = rng.standard_normal((9, 6)), rng.standard_normal((9, 6))
    w, b = 1 + 0.3 * rng.standard_normal(6), rng.standard_normal(6)
    loss = lambda: (dy * B.group_norm(x, 3, w, b, 1e-3, cu, silu)).sum()  # noqa: E731
    got = B.group_norm_backward(x, dy, 3, w, b, 1e-3, cu, silu)
    # a central difference's own error: step^2 f''' / 6, below 1e-6 here (rstd up to 30 in the one-row sequence)
    for t, g in zip((x, w, b), got):
        np.testing.assert_allclose(_central(loss, t), g, rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("causal", [False, True])
def test_diff_attention_gradient_against_differences(causal):
    rng = np.random.default_rng(1)
    cq, ck = [0, 4, 6, 6, 8], [0, 3, 3, 5, 6]
    q, k = rng.standard_normal((8, 8, 64)), rng.standard_normal((6, 4, 64))
    v, lam = rng.standard_normal((6, 2, 128)), rng.uniform(0.2, 0.8, 4)
    dout = rng.standard_normal((8, 4, 128))
    f = lambda: (dout * B.diff_attention(q, k, v, lam, cq, ck, causal=causal)["out"]).sum()  # noqa: E731
    got = B.diff_attention(q, k, v, lam, cq, ck, causal=causal, dout=dout)
    for name, t in (("dq", q), ("dk", k), ("dv", v)):
        at = [tuple(rng.integers(0, n) for n in t.shape) for _ in range(40)]
        for i in at:
            keep, step = t[i], 1e-5
            t[i] = keep + step
            a = f()
            t[i] = keep - step
            b = f()
            t[i] = keep
            assert abs((a - b) / (2 * step) - got[name][i]) < 1e-6, (name, i)
    np.testing.assert_allclose(_central(f, lam), got["dlam"], rtol=1e-6, atol=1e-6)


def test_offsets_are_checked(pkg):
    f = pkg.block_ops._offsets
    assert list(f([0, 3, 3, 7], 7, "cu")) == [0, 3, 3, 7]
    assert list(f(np.array([0, 7], np.int64), 7, "cu")) == [0, 7]
    assert list(f(torch.tensor([0, 7]), 7, "cu")) == [0, 7]
    for bad in ([0], [], [0, 6], [0, 8], [1, 7], [0, 5, 4, 7], [0, -1, 7], [0, 2**32 + 1, 7]):
        with pytest.raises(ValueError):
            f(bad, 7, "cu")
    with pytest.raises((TypeError, ValueError)):
        f([0, 3.5, 7], 7, "cu")
    with pytest.raises(ValueError):
        f(torch.tensor([0.0, 7.0]), 7, "cu")
    with pytest.raises(ValueError):
        f(torch.tensor([[0, 7]]), 7, "cu")


def test_group_norm_refusals(pkg):
    x = torch.zeros(6, 8)
    f = pkg.sparse_group_norm
    with pytest.raises(ValueError, match="CUDA"):
        f(x, 4)
    with pytest.raises(TypeError):
        f(x.double(), 4)
    with pytest.raises(ValueError, match="groups"):
        f(x, 3)
    with pytest.raises(ValueError, match="groups"):
        f(x, 0)
    with pytest.raises(ValueError):
        f(x[0], 4)
    with pytest.raises(ValueError, match="weight"):
        f(x, 4, torch.zeros(7))
    with pytest.raises(TypeError, match="bias"):
        f(x, 4, None, torch.zeros(8, dtype=torch.float16))
    with pytest.raises(TypeError, match="one dtype"):
        f(x.half(), 4, torch.zeros(8), torch.zeros(8, dtype=torch.float16))
    for eps in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="eps"):
            f(x, 4, eps=eps)
    with pytest.raises(ValueError, match="end at"):
        f(x, 4, cu_seqlens=[0, 5])


class _Recorder:
    """An engine that keeps what its calls pass: the values behind the given arguments, read as dense f32."""

    def __init__(self, count, at):
        self.count, self.at, self.seen = count, at, []

    def call(self, name, *args):
        read = lambda p: np.ctypeslib.as_array((ctypes.c_float * self.count).from_address(p)).copy()  # noqa: E731
        self.seen.append((name, *(None if args[i] is None else read(args[i]) for i in self.at[name])))


@pytest.mark.parametrize("grad", [False, True])
def test_group_norm_passes_dense_weights(pkg, monkeypatch, grad):
    """The library reads C consecutive values of weight and bias, so strided and expanded ones are copied, in both
    directions.  (Their storages hold more than C values: the reads here stay in range whatever is passed.)"""
    ops, c = pkg.block_ops, 8
    x, dy = torch.randn(6, c), torch.ones(6, c)
    table = torch.randn(2 * c, 3)
    w, b = table[:c, 1], table.view(-1)[4:5].expand(c)
    engine = _Recorder(c, {"sc_group_norm": (2, 3), "sc_group_norm_backward": (3, 4)})
    monkeypatch.setattr(ops, "get_engine", lambda device: engine)
    cu = ops._offsets([0, 6], 6, "cu")
    if grad:
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        torch.autograd.grad(ops._GroupNorm.apply(*leaves, 4, 1e-5, cu, True), leaves, dy)
    else:
        ops._gn_forward(x, 4, w, b, 1e-5, cu, True, None, False)
    assert [s[0] for s in engine.seen] == ["sc_group_norm", "sc_group_norm_backward"][:1 + grad]
    for _, gw, gb in engine.seen:
        np.testing.assert_array_equal(gw, w.numpy())
        np.testing.assert_array_equal(gb, b.numpy())


def test_dual_tensors_take_part_in_autograd(pkg):
    """They go to the autograd function, as tensors that require grad do (which refuses them: see the GPU tests)."""
    from torch.autograd import forward_ad
    wants, x = pkg.block_ops._wants_grad, torch.zeros(2, 2)
    assert not wants(x, None, 0.5) and wants(x, torch.zeros(1, requires_grad=True), None)
    with torch.no_grad():
        assert not wants(torch.zeros(1, requires_grad=True))
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones(2, 2))
        assert not wants(x) and wants(None, dual)


def test_engine_synchronizes_the_device_once_operators_ran(pkg, monkeypatch):
    """The operators' handle is read after all streams, on the caller's stream; an engine that ran none waits for its
    own stream alone, as before."""
    import threading
    done = []

    class Library:
        def __getattr__(self, name):
            return lambda *args: done.append((name, *args)) or 0
    engine = object.__new__(pkg.Engine)
    engine.lib, engine.handle, engine._op_handle = Library(), None, "ops"
    engine.device, engine._op_lock, engine._op_used = torch.device("cuda", 0), threading.Lock(), False
    current = ["a"]
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: current[0], raising=False)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device: done.append(("device", device)))
    engine.synchronize()
    assert done == [("sc_synchronize", None)]
    engine.call("sc_group_norm", 1)
    current[0] = "b"
    engine.call("sc_group_norm", 2)
    current[0] = "c"
    done.clear()
    engine.synchronize()
    assert done == [("sc_synchronize", None), ("device", engine.device), ("sc_set_stream", "ops", "c"),
                    ("sc_synchronize", "ops")]
    done.clear()
    engine.close()  # not on a stream that its caller may have destroyed
    assert done == [("sc_set_stream", "ops", None), ("sc_destroy", "ops")] and engine._op_handle is None


def test_diff_attention_refusals(pkg):
    h = torch.bfloat16
    q, k, v = torch.zeros(5, 8, 64, dtype=h), torch.zeros(7, 4, 64, dtype=h), torch.zeros(7, 2, 128, dtype=h)
    f = lambda q=q, k=k, v=v, lam=0.5, a=(0, 5), b=(0, 7), **kw: pkg.sparse_diff_attention(q, k, v, lam, a, b, **kw)  # noqa: E731
    with pytest.raises(ValueError, match="CUDA"):
        f()
    with pytest.raises(TypeError):
        f(q=q.float())
    with pytest.raises(TypeError, match="one dtype"):
        f(k=k.half())
    with pytest.raises(ValueError):
        f(q=torch.zeros(5, 8, 32, dtype=h))
    with pytest.raises(ValueError):
        f(v=torch.zeros(7, 2, 64, dtype=h))
    with pytest.raises(ValueError, match="H a multiple"):
        f(q=torch.zeros(5, 6, 64, dtype=h))  # 3 heads over 2
    with pytest.raises(ValueError, match="H a multiple"):
        f(q=torch.zeros(5, 9, 64, dtype=h))
    with pytest.raises(ValueError, match="H a multiple"):
        f(v=torch.zeros(6, 2, 128, dtype=h))
    with pytest.raises(ValueError, match="lam"):
        f(lam=torch.zeros(3, dtype=h))
    with pytest.raises(ValueError, match="lam"):
        f(lam=torch.zeros(1, 4, dtype=h))
    with pytest.raises(TypeError, match="lam"):
        f(lam=torch.zeros(4, dtype=torch.float64))
    with pytest.raises(ValueError, match="end at"):
        f(a=(0, 4))
    with pytest.raises(ValueError, match="same count"):
        f(b=(0, 3, 7))
    with pytest.raises(ValueError, match="pass cu_seqlens_kv"):
        f(b=None)
    for s in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="scale"):
            f(scale=s)


def test_null_handles_are_refused(pkg):
    L, st = pkg._lib.lib(), pkg._lib.SC_EINVAL
    assert L.sc_group_norm(None, None, 0, None, None, None, None, None, 1, 8, 4, 1e-5, 0, 1, 1) == st
    assert L.sc_group_norm_backward(None, None, 0, None, None, None, None, None, None, None, None, 1, 8, 4, 0, 1,
                                    1) == st
    assert L.sc_diff_attention(None, None) == st
    assert L.sc_diff_attention_backward(None, None) == st
