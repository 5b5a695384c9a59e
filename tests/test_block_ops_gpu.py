"""Group norm and differential attention on the GPU, against float64 restatements.

A rounding to type t is off by at most u = finfo(t).eps / 2 of the value.
Group norm rounds once, its f32 arithmetic (some tens of roundings of 2^-24 and
a sigmoid good to 2^-20) stays below 1e-5 of the terms: the relative L2 error is
below u + 1e-5.  Differential attention is held elementwise to the bound that
``oracle.block_ref`` derives for its roundings (weights, score gradients, kept
product, outputs), and over a whole tensor to 2u + 2e-4 relative L2: two to
three independent roundings of at most u.
"""
import numpy as np
import pytest
import torch

from oracle import block_ref as B

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def _f64(t):
    return t.detach().double().cpu().numpy()


def _rel(a, b):
    return float(np.linalg.norm(a - b) / max(np.linalg.norm(b), 1e-30))


def _half(t):
    return torch.finfo(t).eps / 2


def _cu(lens):
    return [0] + np.cumsum(lens).tolist()


# ------------------------------------------------------------------ group norm
def _gn_inputs(cuda, n, c, dtype, wdtype, seed, offset=1.0):
    rng = np.random.default_rng(seed)
    mk = lambda a, t: torch.from_numpy(a.astype(np.float32)).to(cuda, t)  # noqa: E731
    x = rng.standard_normal((n, c)) * rng.uniform(0.5, 2, c) + offset * rng.standard_normal(c)
    return (mk(x, dtype), mk(1 + 0.3 * rng.standard_normal(c), wdtype), mk(0.3 * rng.standard_normal(c), wdtype),
            mk(rng.standard_normal((n, c)), dtype))


def _gn_check(pkg, cuda, lens, c, groups, dtype, wdtype, silu, seed=0, eps=1e-5):
    cu = _cu(lens)
    x, w, b, dy = _gn_inputs(cuda, cu[-1], c, dtype, wdtype, seed)
    for t in (x, w, b):
        t.requires_grad_()
    y = pkg.sparse_group_norm(x, groups, w, b, eps, cu_seqlens=cu, silu=silu)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    with torch.no_grad():
        assert torch.equal(pkg.sparse_group_norm(x, groups, w, b, eps, cu_seqlens=cu, silu=silu), y)
    args = (groups, _f64(w), _f64(b), eps, cu, silu)
    ry = B.group_norm(_f64(x), *args)
    rx, rw, rb = B.group_norm_backward(_f64(x), _f64(dy), *args)
    for got, ref, t in ((y, ry, dtype), (dx, rx, dtype), (dw, rw, wdtype), (db, rb, wdtype)):
        assert got.dtype == t and got.shape == ref.shape
        assert _rel(_f64(got), ref) < (_half(t) if t != FP else 0) + 1e-5, (t, _rel(_f64(got), ref))
    for lo, hi in zip(cu, cu[1:]):
        if hi > lo:
            assert _rel(_f64(y[lo:hi]), ry[lo:hi]) < (_half(dtype) if dtype != FP else 0) + 1e-5


@pytest.mark.parametrize("dtype,wdtype", [(FP, FP), (BF, BF), (BF, FP), (HF, HF), (HF, FP)])
@pytest.mark.parametrize("lens,c,groups", [
    ([300], 64, 32), ([1], 32, 8), ([2, 1, 0, 700, 33], 64, 4), ([129, 257], 36, 9), ([40, 3], 7, 7), ([65], 6, 1),
    ([1000, 1500], 256, 32), ([17, 90], 4096, 32), ([50], 4095, 5), ([9001], 96, 3), ([30], 4096, 4096),
    ([700], 1024, 1024)])
def test_group_norm(pkg, cuda, dtype, wdtype, lens, c, groups):
    _gn_check(pkg, cuda, lens, c, groups, dtype, wdtype, silu=True)


@pytest.mark.parametrize("lens,c,groups", [([513, 5], 128, 32), ([3000], 24, 12)])
def test_group_norm_without_activation(pkg, cuda, lens, c, groups):
    _gn_check(pkg, cuda, lens, c, groups, BF, BF, silu=False, seed=3)
    _gn_check(pkg, cuda, lens, c, groups, FP, FP, silu=False, seed=4, eps=1e-2)


def test_group_norm_many_sequences(pkg, cuda):
    """More sequences than travel in a kernel's parameters, some without rows."""
    rng = np.random.default_rng(5)
    _gn_check(pkg, cuda, rng.integers(0, 9, 700).tolist(), 32, 8, BF, FP, silu=True)


def test_group_norm_large(pkg, cuda):
    _gn_check(pkg, cuda, [40000, 123, 60000], 64, 16, BF, FP, silu=True, seed=6)


@pytest.mark.parametrize("dtype,wdtype,lens,c,groups,silu", [
    (BF, FP, [20011, 1, 0, 30007, 123, 15003], 256, 32, True),  # vectors of one group
    (BF, BF, [105003], 96, 3, True), (BF, BF, [60001, 45007], 96, 8, False),  # 504 of 512 threads have a column
    (HF, HF, [50021, 30011], 128, 32, True), (HF, FP, [80033], 128, 4, False),
    (FP, FP, [80033], 64, 16, True), (FP, FP, [50021, 2, 30011], 64, 32, True), (FP, FP, [80033], 64, 64, False),
    (BF, FP, [3001, 1999], 2048, 16, True), (BF, BF, [2000, 707], 4096, 32, True)])
def test_group_norm_through_the_ring(pkg, cuda, dtype, wdtype, lens, c, groups, silu):
    """Rows through the ring of bulk copies, forward and backward, last blocks short: all rows and gradients."""
    vectors = c * torch.finfo(dtype).bits // 128
    slots = 2 * torch.cuda.get_device_properties(cuda).multi_processor_count
    assert sum(lens) >= slots * 8 * (512 // vectors)  # chunks of eight rows a thread at least
    _gn_check(pkg, cuda, lens, c, groups, dtype, wdtype, silu, seed=70)


@pytest.mark.parametrize("dtype,c,groups,wide", [(BF, 64, 16, 16), (BF, 72, 8, 8), (HF, 66, 11, 3), (FP, 64, 32, 4)])
def test_group_norm_long_rows_without_the_ring(pkg, cuda, dtype, c, groups, wide):
    """Rows apart, as in a slice of a fused buffer, also of no whole 16-byte words: several chunks of many rows."""
    cu = _cu([70001, 30, 29007])
    x, w, b, dy = _gn_inputs(cuda, cu[-1], c, dtype, FP, 71)
    x = torch.cat((dy[:, :wide], x), 1)[:, wide:].requires_grad_()
    w.requires_grad_(), b.requires_grad_()
    y = pkg.sparse_group_norm(x, groups, w, b, cu_seqlens=cu, silu=True)
    got = (y, *torch.autograd.grad(y, (x, w, b), dy))
    args = (groups, _f64(w), _f64(b), 1e-5, cu, True)
    ref = (B.group_norm(_f64(x), *args), *B.group_norm_backward(_f64(x), _f64(dy), *args))
    for g, r, t in zip(got, ref, (dtype, dtype, FP, FP)):
        assert _rel(_f64(g), r) < (_half(t) if t != FP else 0) + 1e-5, (t, _rel(_f64(g), r))


def test_group_norm_through_the_ring_in_place(pkg, cuda):
    for dtype, c in ((BF, 256), (FP, 64)):
        x, w, b, _ = _gn_inputs(cuda, 80033, c, dtype, FP, 72)
        ref = pkg.sparse_group_norm(x, 16, w, b, silu=True, cu_seqlens=[0, 50001, 80033])
        assert pkg.sparse_group_norm(x, 16, w, b, silu=True, cu_seqlens=[0, 50001, 80033], out=x) is x
        assert torch.equal(x, ref)


def test_group_norm_without_weights(pkg, oracle, cuda):
    x, _, b, dy = _gn_inputs(cuda, 400, 48, FP, FP, 7)
    y = pkg.sparse_group_norm(x, 6)
    assert _rel(_f64(y), B.group_norm(_f64(x), 6, None, None, 1e-5, [0, 400], False)) < 1e-5
    b.requires_grad_()
    y = pkg.sparse_group_norm(x, 6, None, b, silu=True)
    db, = torch.autograd.grad(y, (b,), dy)
    ref = B.group_norm_backward(_f64(x), _f64(dy), 6, None, _f64(b), 1e-5, [0, 400], True)[2]
    assert _rel(_f64(db), ref) < 1e-5


def test_group_norm_far_from_zero(pkg, cuda):
    """Means 1000 deviations from zero, and a first row far from the rest: the
    mean is good to some 2^-24 of itself (1000 * 2^-24 * a few = 3e-4 of a
    deviation), and so is xhat."""
    x, _, _, _ = _gn_inputs(cuda, 5000, 64, FP, FP, 8, offset=0.0)
    x += 1000.0
    y = pkg.sparse_group_norm(x, 8)
    assert _rel(_f64(y), B.group_norm(_f64(x), 8, None, None, 1e-5, [0, 5000], False)) < 3e-4
    x -= 1000.0
    x[0] += 3e4
    y = pkg.sparse_group_norm(x, 8)
    assert _rel(_f64(y), B.group_norm(_f64(x), 8, None, None, 1e-5, [0, 5000], False)) < 1e-5


def test_group_norm_rows_apart_and_in_place(pkg, cuda):
    wide, w, b, dy = _gn_inputs(cuda, 333, 200, BF, BF, 9)
    x = wide[:, 8:72]
    w, b = w[:64].contiguous(), b[:64].contiguous()
    ref = pkg.sparse_group_norm(x.contiguous(), 16, w, b, silu=True)
    assert torch.equal(pkg.sparse_group_norm(x, 16, w, b, silu=True), ref)
    assert torch.equal(pkg.sparse_group_norm(wide[:, 3:67], 16, w, b, silu=True),
                       pkg.sparse_group_norm(wide[:, 3:67].contiguous(), 16, w, b, silu=True))
    t = x.t().contiguous().t()  # channels apart: a copy is taken
    assert torch.equal(pkg.sparse_group_norm(t, 16, w, b, silu=True), ref)
    # gradients of the slice, with a broadcast gradient
    xs = x.detach().requires_grad_()
    gx, = torch.autograd.grad(pkg.sparse_group_norm(xs, 16, w, b, silu=True), (xs,), dy[:1, :64].expand(333, 64))
    xc = x.contiguous().detach().requires_grad_()
    gc, = torch.autograd.grad(pkg.sparse_group_norm(xc, 16, w, b, silu=True), (xc,),
                              dy[:1, :64].expand(333, 64).contiguous())
    assert torch.equal(gx, gc)
    xc = xc.detach()
    out = pkg.sparse_group_norm(xc, 16, w, b, silu=True, out=xc)
    assert out is xc and torch.equal(xc, ref)
    with pytest.raises(ValueError, match="overlaps"):
        pkg.sparse_group_norm(wide.view(-1)[: 332 * 200].view(-1, 200), 8, out=wide.view(-1)[200: 333 * 200].view(-1, 200))
    with pytest.raises(ValueError, match="autograd"):
        pkg.sparse_group_norm(xs, 16, w, b, out=xc)
    with pytest.raises(ValueError, match="out must"):
        pkg.sparse_group_norm(xc, 16, w, b, out=xc.float())


@pytest.mark.parametrize("dtype", [FP, BF])
def test_group_norm_weights_apart(pkg, cuda, dtype):
    """A column of a table and an expanded single value as weight or bias, with and without gradients: as the dense ones."""
    x, w, b, dy = _gn_inputs(cuda, 333, 64, dtype, FP, 12)
    table = torch.stack((b, w, b), 1)
    col, one = table[:, 1], w[5:6].expand(64)
    for weight, bias in ((col, one), (one, table[:, 0]), (col, None), (None, one)):
        dense = [None if t is None else t.contiguous() for t in (weight, bias)]
        ref = pkg.sparse_group_norm(x, 16, *dense, silu=True)
        assert torch.equal(pkg.sparse_group_norm(x, 16, weight, bias, silu=True), ref)
        given = []
        for pair in (dense, (weight, bias)):
            leaves = [t.detach().requires_grad_() for t in (x, *pair) if t is not None]
            vectors = iter(leaves[1:])
            y = pkg.sparse_group_norm(leaves[0], 16, *(None if t is None else next(vectors) for t in pair), silu=True)
            given.append((y, *torch.autograd.grad(y, leaves, dy)))
        assert torch.equal(given[0][0], ref)
        assert all(torch.equal(p, r) for p, r in zip(*given))


def test_group_norm_of_nothing(pkg, cuda):
    x = torch.zeros(0, 32, device=cuda, dtype=BF, requires_grad=True)
    w = torch.ones(32, device=cuda, requires_grad=True)
    y = pkg.sparse_group_norm(x, 4, w, cu_seqlens=[0, 0, 0])
    assert y.shape == (0, 32)
    dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
    assert dx.shape == (0, 32) and torch.count_nonzero(dw) == 0


def test_group_norm_keeps_sequences_and_groups_apart(pkg, cuda):
    x, w, b, _ = _gn_inputs(cuda, 700, 64, BF, BF, 10)
    cu = [0, 300, 301, 700]
    ref = pkg.sparse_group_norm(x, 8, w, b, cu_seqlens=cu)
    x[300, 3] = float("nan")
    x[400, 20] = float("inf")
    got = pkg.sparse_group_norm(x, 8, w, b, cu_seqlens=cu)
    assert torch.equal(got[:300], ref[:300])
    assert torch.equal(got[300, 8:], ref[300, 8:]) and got[300, :8].isnan().all()
    assert torch.equal(got[301:, :16], ref[301:, :16]) and torch.equal(got[301:, 24:], ref[301:, 24:])


def test_group_norm_past_32_bit_offsets(pkg, cuda):
    """2.2e9 values: the last sequence lies past 2^31 elements."""
    n, c = 17_200_000, 128
    x = torch.full((n, c), 0.5, dtype=BF, device=cuda)
    tail, w, b, _ = _gn_inputs(cuda, 900, c, BF, BF, 11)
    x[-900:] = tail
    y = pkg.sparse_group_norm(x, 32, w, b, cu_seqlens=[0, 7, n - 900, n], silu=True, out=x)
    ref = B.group_norm(_f64(tail), 32, _f64(w), _f64(b), 1e-5, [0, 900], True)
    assert _rel(_f64(y[-900:]), ref) < _half(BF) + 1e-5


# ------------------------------------------------------ differential attention
def _da_inputs(cuda, nq, nkv, heads, kv_heads, dtype, seed, spread=1.5):
    rng = np.random.default_rng(seed)
    mk = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).to(cuda)  # noqa: E731
    return ((spread * mk(nq, 2 * heads, 64)).to(dtype), mk(nkv, 2 * kv_heads, 64).to(dtype),
            mk(nkv, kv_heads, 128).to(dtype),
            torch.from_numpy(rng.uniform(0.2, 0.8, heads).astype(np.float32)).to(cuda), mk(nq, heads, 128).to(dtype))


def _close(got, ref, name, u):
    g, r, bound = _f64(got), ref[name], ref[name + "_bound"]
    over = np.abs(g - r) - bound
    tiny = 2.0 ** -24 if u < 2.0 ** -9 else 0.0  # f16 results below its normal range are rounded in absolute steps
    assert np.isfinite(g).all()
    assert over.max(initial=-1) <= tiny, (name, np.unravel_index(over.argmax(), over.shape), over.max())
    if np.linalg.norm(r) > 0:
        assert _rel(g, r) < 2 * u + 2e-4, (name, _rel(g, r))


def _da_check(pkg, cuda, lq, lk, heads, kv_heads, dtype, causal, seed=0, train=True, scale=None, spread=1.5, gain=1.0):
    cq, ck = _cu(lq), _cu(lk)
    q, k, v, lam, dout = _da_inputs(cuda, cq[-1], ck[-1], heads, kv_heads, dtype, seed, spread)
    dout = dout * gain
    with torch.no_grad():
        out = pkg.sparse_diff_attention(q, k, v, lam, cq, ck, scale, causal)
    u = _half(dtype)
    ref = B.diff_attention(_f64(q), _f64(k), _f64(v), _f64(lam), cq, ck, 0.125 if scale is None else scale, causal,
                           _f64(dout) if train else None, u)
    assert out.dtype == dtype and out.shape == (cq[-1], heads, 128)
    _close(out, ref, "out", u)
    see = np.zeros(cq[-1], bool)
    for b in range(len(lq)):
        see[cq[b]:cq[b + 1]] = (np.arange(lq[b]) + lk[b] - lq[b] >= 0) if causal else lk[b] > 0
    see &= np.concatenate([np.full(n, m > 0) for n, m in zip(lq, lk)]) if cq[-1] else True
    assert torch.count_nonzero(out[torch.from_numpy(~see).to(cuda)]) == 0
    if not train:
        return
    leaves = [t.requires_grad_() for t in (q, k, v, lam)]
    got_out = pkg.sparse_diff_attention(q, k, v, lam, cq, ck, scale, causal)
    _close(got_out, ref, "out", u)
    for name, g, t in zip(("dq", "dk", "dv", "dlam"), torch.autograd.grad(got_out, leaves, dout), leaves):
        assert g.dtype == t.dtype and g.shape == t.shape
        if name == "dlam":
            assert (np.abs(_f64(g) - ref["dlam"]) <= ref["dlam_bound"] + 1e-6).all()
        else:
            _close(g, ref, name, u)


SHAPES = [([300], [300]), ([1], [1]), ([128], [128]), ([129, 1, 257, 64], [129, 1, 257, 64]),
          ([70, 0, 200, 33, 5], [130, 9, 1, 0, 300]), ([1, 1, 1], [700, 1, 130]), ([2, 127], [1000, 126])]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lq,lk", SHAPES)
def test_diff_attention(pkg, cuda, dtype, causal, lq, lk):
    _da_check(pkg, cuda, lq, lk, 4, 2, dtype, causal, seed=sum(lq))


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 1), (6, 2), (8, 1), (5, 5), (40, 1)])
def test_diff_attention_heads(pkg, cuda, heads, kv_heads):
    _da_check(pkg, cuda, [150, 40], [150, 40], heads, kv_heads, BF, True, seed=heads)
    _da_check(pkg, cuda, [1, 3], [400, 90], heads, kv_heads, HF, True, seed=heads, train=False)


@pytest.mark.parametrize("lk", [1, 63, 64, 65, 127, 128, 129, 1023, 5000])
def test_diff_attention_single_token(pkg, cuda, lk):
    _da_check(pkg, cuda, [1], [lk], 8, 4, BF, True, seed=lk, train=False)
    _da_check(pkg, cuda, [1, 1, 1], [lk, 0, 2 * lk], 2, 2, HF, False, seed=lk, train=False)


def test_diff_attention_longer(pkg, cuda):
    _da_check(pkg, cuda, [1100, 700], [1100, 700], 2, 1, BF, False, seed=20)
    _da_check(pkg, cuda, [1500], [1300], 2, 2, HF, True, seed=21)
    _da_check(pkg, cuda, [400], [3000], 2, 1, BF, True, seed=22)


def test_diff_attention_large_scores(pkg, cuda):
    """Scores of deviation 20: the softmax picks single keys, and the running maximum moves."""
    _da_check(pkg, cuda, [260, 30], [900, 300], 4, 2, BF, False, seed=23, spread=20.0, train=False)
    _da_check(pkg, cuda, [200], [200], 2, 2, HF, True, seed=24, scale=0.3, train=False)


def test_diff_attention_scales_and_gains(pkg, cuda):
    """The ends of the scale's range (at 2^-20 every weight is 1 / n), and gradients as a loss scale makes them."""
    for dtype in (BF, HF):
        _da_check(pkg, cuda, [150, 40], [150, 90], 2, 1, dtype, True, seed=32, scale=2.0 ** -20, train=False)
        _da_check(pkg, cuda, [150, 40], [150, 90], 2, 1, dtype, False, seed=33, scale=2.0, spread=0.1)
        _da_check(pkg, cuda, [150, 40], [150, 90], 2, 1, dtype, True, seed=34, gain=64.0)
        _da_check(pkg, cuda, [150, 40], [150, 90], 2, 1, dtype, True, seed=35, gain=2.0 ** -6)
    cu = [0, 100]
    q, k, v, lam, dout = _da_inputs(cuda, 100, 100, 2, 2, HF, 36)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    got = torch.autograd.grad(pkg.sparse_diff_attention(q, k, v, lam, cu, scale=2.0 ** -20), leaves, dout)
    ref = B.diff_attention(_f64(q), _f64(k), _f64(v), _f64(lam), cu, scale=2.0 ** -20, dout=_f64(dout), u=_half(HF))
    _close(got[2], ref, "dv", _half(HF))


def _da_small_gradients(pkg, cuda, nq, nkv, gain, seed, heads=2, kv_heads=1, parts=((0, None),)):
    """f16 gradients of one sequence where they, the weights or the score gradients are small or large: elementwise
    as ever, and over the rows of each part the relative L2 bound of this file beside the absolute step of results
    below the normal range (half of 2^-24 an element)."""
    q, k, v, lam, dout = _da_inputs(cuda, nq, nkv, heads, kv_heads, HF, seed)
    dout = (dout.float() * gain).to(HF)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    got = torch.autograd.grad(pkg.sparse_diff_attention(q, k, v, lam, [0, nq], [0, nkv]), leaves, dout)
    ref = B.diff_attention(_f64(q), _f64(k), _f64(v), _f64(lam), [0, nq], [0, nkv], dout=_f64(dout), u=_half(HF))
    for name, g in zip(("dq", "dk", "dv"), got):
        err = np.abs(_f64(g) - ref[name])
        assert np.isfinite(err).all() and (err <= ref[name + "_bound"] + 2.0 ** -25).all(), name
        for first, step in parts if name == "dq" else ((0, None),):
            e, r = err[first::step], ref[name][first::step]
            most = (2 * _half(HF) + 2e-4) * np.linalg.norm(r) + 2.0 ** -25 * r.size ** 0.5
            assert np.linalg.norm(e) <= most, (name, np.linalg.norm(e), most)


@pytest.mark.parametrize("gain", [1.0, 2.0 ** -7, 2.0 ** -10, 2.0 ** -14])
def test_diff_attention_f16_small_gradients(pkg, cuda, gain):
    """dout as a mean over many values makes it, weights of 1 / 8192."""
    _da_small_gradients(pkg, cuda, 256, 8192, gain, 60)


def test_diff_attention_f16_small_weights(pkg, cuda):
    """Weights of 5e-6, below f16's normal range: dv is made from them."""
    _da_small_gradients(pkg, cuda, 64, 200_000, 64.0, 61, heads=1)


def test_diff_attention_f16_large_gradients(pkg, cuda):
    """dP - delta past 65,504, as under a loss scale, with gradients that fit."""
    _da_small_gradients(pkg, cuda, 4, 8, 2.0 ** 13, 62)


def test_diff_attention_f16_rows_of_other_size(pkg, cuda):
    """Rows whose dout is 2^-10 of the others' keep their dq."""
    gain = torch.ones(256, 1, 1, device=cuda)
    gain[::2] = 2.0 ** -10
    _da_small_gradients(pkg, cuda, 256, 8192, gain, 63, parts=((0, 2), (1, 2)))


@pytest.mark.parametrize("nq", [1, 150])
def test_diff_attention_f16_weights_far_below_the_largest(pkg, cuda, nq):
    """500 keys of weight 2^-25 to 2^-26 beside one of weight 1 whose values are zero: all of the output comes from
    them.  A weight is off by at most 2^-32 of the row's largest (half a step of f16's smallest numbers, weights
    written 2^7 times larger)."""
    rng = np.random.default_rng(65)
    q = torch.ones(nq, 2, 64, dtype=HF, device=cuda)
    k = torch.from_numpy(rng.uniform(-1.14, -1.08, (500, 2, 1)).astype(np.float32)).to(cuda, HF).repeat(1, 1, 64)
    k[37] = 1.1
    v = torch.full((500, 1, 128), 1000.0, dtype=HF, device=cuda)
    v[37] = 0
    cu_q, cu_kv = [0, nq], [0, 500]
    got = pkg.sparse_diff_attention(q, k, v, -1.0, cu_q, cu_kv)
    ref = B.diff_attention(_f64(q), _f64(k), _f64(v), np.array([-1.0]), cu_q, cu_kv, u=_half(HF))
    assert ref["out"].min() > 0.01
    assert (np.abs(_f64(got) - ref["out"]) <= ref["out_bound"] + 2 * 2.0 ** -32 * 499 * 1000).all()


def test_diff_attention_f16_large_lam(pkg, cuda):
    """lam far from 1 scales one map's score gradients and its part of the weights."""
    for lam in (40.0, -0.01, 0.0):
        q, k, v, _, dout = _da_inputs(cuda, 200, 300, 4, 2, HF, 64)
        leaves = [t.requires_grad_() for t in (q, k, v)]
        got = torch.autograd.grad(pkg.sparse_diff_attention(q, k, v, lam, [0, 200], [0, 300]), leaves, dout)
        ref = B.diff_attention(_f64(q), _f64(k), _f64(v), np.full(4, lam), [0, 200], [0, 300], dout=_f64(dout),
                               u=_half(HF))
        for name, g in zip(("dq", "dk", "dv"), got):
            _close(g, ref, name, _half(HF))


def test_diff_attention_prefill_beside_single_tokens(pkg, cuda):
    """Sequences whose keys are cut into ranges beside some whose are not."""
    for dtype in (BF, HF):
        _da_check(pkg, cuda, [1, 300, 2, 40], [5000, 300, 9000, 100], 4, 2, dtype, True, seed=37, train=False)
    _da_check(pkg, cuda, [1, 200, 2], [2500, 200, 1200], 2, 1, BF, True, seed=38)


def test_diff_attention_many_sequences(pkg, cuda):
    rng = np.random.default_rng(25)
    lq, lk = rng.integers(0, 6, 300).tolist(), rng.integers(0, 40, 300).tolist()
    _da_check(pkg, cuda, lq, lk, 2, 1, BF, True, seed=26)


def test_diff_attention_lam_forms(pkg, cuda):
    q, k, v, _, dout = _da_inputs(cuda, 200, 200, 4, 4, BF, 27)
    cu = [0, 200]
    each = torch.full((4,), 0.5, device=cuda)
    ref = pkg.sparse_diff_attention(q, k, v, each, cu)
    for lam in (0.5, torch.tensor(0.5, device=cuda), torch.full((1,), 0.5, device=cuda, dtype=BF), each.to(BF)):
        assert torch.equal(pkg.sparse_diff_attention(q, k, v, lam, cu), ref)
    each.requires_grad_()
    g, = torch.autograd.grad(pkg.sparse_diff_attention(q, k, v, each, cu), (each,), dout)
    one = torch.tensor(0.5, device=cuda, requires_grad=True)
    g1, = torch.autograd.grad(pkg.sparse_diff_attention(q, k, v, one, cu), (one,), dout)
    assert g1.shape == () and abs(g1.item() - g.double().sum().item()) <= 1e-5 * g.double().abs().sum().item()
    q.requires_grad_()
    gq, = torch.autograd.grad(pkg.sparse_diff_attention(q, k, v, 0.5, cu), (q,), dout)
    assert gq.shape == q.shape


def test_diff_attention_only_asked_gradients(pkg, cuda):
    q, k, v, lam, dout = _da_inputs(cuda, 150, 150, 2, 2, BF, 28)
    cu = [0, 60, 150]
    leaves = [t.requires_grad_() for t in (q, k, v, lam)]
    full = torch.autograd.grad(pkg.sparse_diff_attention(q, k, v, lam, cu), leaves, dout)
    for i in range(4):
        for t in leaves:
            t.requires_grad_(False)
        leaves[i].requires_grad_()
        g, = torch.autograd.grad(pkg.sparse_diff_attention(q, k, v, lam, cu), (leaves[i],), dout)
        assert torch.equal(g, full[i])


def test_diff_attention_rows_apart(pkg, cuda):
    """q, k and v as slices of one fused projection, read in place; other layouts are copied."""
    rng = np.random.default_rng(29)
    fused = torch.from_numpy(rng.standard_normal((210, 1536)).astype(np.float32)).to(cuda, BF)
    q = fused[:, :512].unflatten(1, (8, 64))
    k, v = fused[:, 512:1024].unflatten(1, (8, 64)), fused[:, 1024:].unflatten(1, (4, 128))
    cu = [0, 10, 210]
    ref = pkg.sparse_diff_attention(q.contiguous(), k.contiguous(), v.contiguous(), 0.4, cu, causal=True)
    assert torch.equal(pkg.sparse_diff_attention(q, k, v, 0.4, cu, causal=True), ref)
    swapped = q.transpose(0, 1).contiguous().transpose(0, 1)
    odd = torch.empty(210 * 512 + 1, dtype=BF, device=cuda)[1:].view(210, 8, 64)
    odd.copy_(k)
    assert torch.equal(pkg.sparse_diff_attention(swapped, odd, v, 0.4, cu, causal=True), ref)
    out = torch.empty_like(ref)
    assert pkg.sparse_diff_attention(q, k, v, 0.4, cu, causal=True, out=out) is out and torch.equal(out, ref)
    with pytest.raises(ValueError, match="overlap"):
        pkg.sparse_diff_attention(q, k, v.contiguous(), 0.4, cu, out=fused.view(-1)[:210 * 512].view(210, 4, 128))


def test_diff_attention_sequences_stay_isolated(pkg, cuda):
    """NaN and infinities in another sequence's rows (same key tile) reach neither outputs nor gradients."""
    cu = [0, 200, 500]
    q, k, v, lam, dout = _da_inputs(cuda, 500, 500, 2, 1, BF, 30)
    leaves = [t.requires_grad_() for t in (q, k, v)]

    def run():
        out = pkg.sparse_diff_attention(q, k, v, 0.5, cu)
        return (out, *torch.autograd.grad(out, leaves, dout))
    ref = run()
    with torch.no_grad():
        q[230], k[250], v[201], v[220], dout[210] = (float("nan"), float("inf"), float("nan"), float("-inf"),
                                                     float("nan"))
    for a, b in zip(run(), ref):
        assert torch.equal(a[:200], b[:200])


def _da_plain(q, k, v, lam, cu_q, cu_kv):
    """Float64, no mask; torch's own rules for NaN and infinities."""
    q, k, v, lam = (t.detach().double().cpu() for t in (q, k, v, lam))
    out = torch.zeros(q.shape[0], q.shape[1] // 2, 128, dtype=torch.float64)
    rep = out.shape[1] // v.shape[1]
    for a, b, c, d in zip(cu_q, cu_q[1:], cu_kv, cu_kv[1:]):
        for h in range(out.shape[1] if b > a and d > c else 0):
            g = h // rep
            m = [torch.softmax(q[a:b, 2 * h + i] @ k[c:d, 2 * g + i].T / 8, -1) @ v[c:d, g] for i in (0, 1)]
            out[a:b, h] = m[0] - lam[h] * m[1]
    return out


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("cu_q,cu_kv", [([0, 150, 300], [0, 200, 500]),  # whole sequences
                                        ([0, 1, 2], [0, 700, 5700])])    # keys cut into ranges
@pytest.mark.parametrize("where", ["q", "q1", "k", "v"])
@pytest.mark.parametrize("bad", ["nan", "inf", "-inf"])
def test_diff_attention_nan_and_infinity_reach_their_rows(pkg, cuda, dtype, train, cu_q, cu_kv, where, bad):
    """A NaN or an infinity in a sequence makes the values non-finite that it makes non-finite in float64, and no
    others; the rest is as close as ever (a score of -inf is a weight of 0).  lse goes with its map."""
    q, k, v, lam, _ = _da_inputs(cuda, cu_q[-1], cu_kv[-1], 4, 2, dtype, 50)
    {"q": q[cu_q[1]], "q1": q[cu_q[1], 1], "k": k[cu_kv[1] + 130], "v": v[cu_kv[1] + 130]}[where][..., 5] = float(bad)
    q.requires_grad_(train)
    got = pkg.sparse_diff_attention(q, k, v, lam, cu_q, cu_kv)
    ref = _da_plain(q, k, v, lam, cu_q, cu_kv)
    fin = ref.isfinite()
    assert not fin.all()
    if where == "v":  # the maps' difference of infinities is NaN, as is 0 * inf of a weight that underflows
        assert not fin[cu_q[1]:, :, 5].any()
    out = got.detach().double().cpu()
    assert torch.equal(out.isfinite(), fin)
    assert _rel(out[fin].numpy(), ref[fin].numpy()) < 2 * _half(dtype) + 2e-4
    if train:
        lse = got.grad_fn.saved_tensors[5]  # [2][heads][rows]
        maps = got.grad_fn.saved_tensors[4]
        if where == "v":
            assert lse.isfinite().all()
        else:
            assert torch.equal(lse.isnan(), maps.isnan().all(3).permute(2, 1, 0))
            assert lse.isnan().any() and not lse.isinf().any()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("where", ["q", "q1", "k", "v", "dout"])
@pytest.mark.parametrize("bad", ["nan", "inf"])
def test_diff_attention_nan_and_infinity_reach_their_gradients(pkg, cuda, dtype, where, bad):
    """Every gradient that float64 makes non-finite is non-finite; another sequence's are untouched."""
    cu_q, cu_kv, heads = [0, 150, 300], [0, 200, 500], 4
    q, k, v, lam, dout = _da_inputs(cuda, 300, 500, heads, 2, dtype, 52)
    leaves = [t.requires_grad_() for t in (q, k, v, lam)]
    clean = torch.autograd.grad(pkg.sparse_diff_attention(*leaves, cu_q, cu_kv), leaves, dout)
    with torch.no_grad():
        {"q": q[170], "q1": q[170, 1], "k": k[330], "v": v[330], "dout": dout[170]}[where][..., 5] = float(bad)
    got = torch.autograd.grad(pkg.sparse_diff_attention(*leaves, cu_q, cu_kv), leaves, dout)
    given = [t.detach().double().cpu().requires_grad_() for t in leaves]
    parts = []
    for a, b, c, d in zip(cu_q, cu_q[1:], cu_kv, cu_kv[1:]):
        hs = []
        for h in range(heads):
            m = [torch.softmax(given[0][a:b, 2 * h + i] @ given[1][c:d, 2 * (h // 2) + i].T / 8, -1) for i in (0, 1)]
            hs.append((m[0] - given[3][h] * m[1]) @ given[2][c:d, h // 2])
        parts.append(torch.stack(hs, 1))
    ref = torch.autograd.grad(torch.cat(parts), given, dout.double().cpu())
    for name, g, r, was, first in zip(("q", "k", "v", "lam"), got, ref, clean, (150, 200, 200, 0)):
        fin = g.isfinite().cpu()
        assert not (fin & ~r.isfinite()).any(), (name, int((fin & ~r.isfinite()).sum()))
        assert torch.equal(g[:first], was[:first])


def test_diff_attention_scores_past_the_f16_statistics(pkg, cuda):
    """f16 scores of 7.1e7 before the scale: the backward says NaN where it can not hold the row's log-sum-exp."""
    q = torch.full((40, 2, 64), 1050.0, dtype=HF, device=cuda)
    k, v, dout = q.clone(), torch.randn(40, 1, 128, device=cuda).to(HF), torch.randn(40, 1, 128, device=cuda).to(HF)
    k[7:] *= -1
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = pkg.sparse_diff_attention(*leaves, 0.5, [0, 40], scale=2.0 ** -20)
    assert out.isfinite().all()
    for g in torch.autograd.grad(out, leaves, dout)[1:]:
        assert g.isnan().any()


@pytest.mark.parametrize("dtype", [BF, HF])
def test_diff_attention_without_a_softmax(pkg, cuda, dtype):
    """Scores that are all -inf have no softmax: NaN, for whole sequences and for joined ranges; without keys a row
    stays zero whatever its query holds."""
    for cu_kv in ([0, 3, 203, 203], [0, 700, 5700, 5700]):
        cu_q = [0, 1, 2, 4]
        q, k, v, lam, _ = _da_inputs(cuda, 4, cu_kv[-1], 2, 1, dtype, 51)
        k[:cu_kv[1], :, 9] = -1.0
        q[0, :, 9] = float("inf")
        q[2:] = float("nan")
        for train in (False, True):
            out = pkg.sparse_diff_attention(q.requires_grad_(train), k, v, lam, cu_q, cu_kv)
            assert out[0].isnan().all() and out[1].isfinite().all() and torch.count_nonzero(out[2:]) == 0
            if train:
                lse = out.grad_fn.saved_tensors[5]
                assert lse[..., 0].isnan().all() and lse[..., 1].isfinite().all() and (lse[..., 2:] == np.inf).all()
            q = q.detach()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("nq,nkv", [(0, 70), (70, 0), (0, 0)])
def test_diff_attention_of_nothing(pkg, cuda, dtype, nq, nkv):
    """No queries, or no keys, in the whole call: zeros, and gradients of zero."""
    q, k, v, lam, dout = _da_inputs(cuda, nq, nkv, 4, 2, dtype, 53)
    leaves = [t.requires_grad_() for t in (q, k, v, lam)]
    out = pkg.sparse_diff_attention(*leaves, [0, 0, nq], [0, nkv, nkv], causal=True)
    assert out.shape == (nq, 4, 128) and torch.count_nonzero(out) == 0
    for g, t in zip(torch.autograd.grad(out, leaves, dout), leaves):
        assert g.shape == t.shape and torch.count_nonzero(g) == 0


@pytest.mark.parametrize("heads,kv_heads", [(129, 1), (256, 2), (128, 1)])
def test_diff_attention_more_heads_than_a_tile_has_rows(pkg, cuda, heads, kv_heads):
    _da_check(pkg, cuda, [3, 1, 140], [200, 70, 150], heads, kv_heads, BF, True, seed=54)
    _da_check(pkg, cuda, [2], [700], heads, kv_heads, HF, False, seed=55, train=False)


def test_diff_attention_f16_captured_and_repeated(pkg, cuda):
    """f16 gradients (their factors come from maxima over the call) repeat bit for bit, also from a graph."""
    cu = [0, 40, 41, 300]
    q, k, v, lam, dout = _da_inputs(cuda, 300, 300, 4, 2, HF, 56)
    leaves = [t.requires_grad_() for t in (q, k, v, lam)]

    def run():
        out = pkg.sparse_diff_attention(*leaves, cu, causal=True)
        return [out.detach(), *torch.autograd.grad(out, leaves, dout)]
    s = torch.cuda.Stream(cuda)
    s.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(s):
        run()
    torch.cuda.current_stream(cuda).wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = run()
    for size in (1.0, 2.0 ** -12, 2.0 ** 8):
        with torch.no_grad():
            q.copy_(torch.randn_like(q))
            dout.copy_(size * torch.randn_like(dout))
        g.replay()
        held = [t.clone() for t in got]
        for _ in range(3):
            assert all(torch.equal(a, b) for a, b in zip(held, run()))


def test_diff_attention_past_32_bit_offsets(pkg, cuda):
    """A cache whose last sequence lies past 2^31 elements of k and v."""
    n, hk = 2_150_000, 8
    k = torch.zeros((n, 2 * hk, 64), dtype=BF, device=cuda)
    v = torch.zeros((n, hk, 128), dtype=BF, device=cuda)
    q, kt, vt, lam, _ = _da_inputs(cuda, 2, 700, hk, hk, BF, 31)
    k[-700:], v[-700:] = kt, vt
    out = pkg.sparse_diff_attention(q, k, v, lam, [0, 1, 2], [0, n - 700, n], causal=True)
    ref = pkg.sparse_diff_attention(q[1:], kt, vt, lam, [0, 1], [0, 700], causal=True)
    assert _rel(_f64(out[1:]), _f64(ref)) < 2 * _half(BF)
    assert torch.count_nonzero(out[0]) == 0  # values of zero


def test_refusals_of_the_c_calls(pkg, cuda):
    """What the entry points refuse before any launch, with their reason; the handle stays usable."""
    import ctypes
    L, engine = pkg._lib, pkg.get_engine(cuda)
    x = torch.randn(8, 64, device=cuda)
    y, stats = torch.empty_like(x), torch.empty(16, device=cuda)
    cu = lambda *a: (ctypes.c_int32 * len(a))(*a)  # noqa: E731

    def refused(match, name, *args):
        with pytest.raises(pkg.SparseConvError, match=match):
            engine.call(name, *args)
    gn = lambda x=x.data_ptr(), xs=64, y=y.data_ptr(), cu=cu(0, 8), batch=1, c=64, g=8, eps=1e-5, t=0, wt=0: (  # noqa: E731
        x, xs, None, None, y, None, cu, batch, c, g, eps, 0, t, wt)
    for match, bad in (("dtype", {"t": 9}), ("weight and bias", {"t": 0, "wt": 1}), ("channels", {"c": 4097, "g": 1}),
                       ("channels", {"g": 7}), ("batch", {"batch": 0}), ("cu_seqlens", {"cu": None}),
                       ("non-decreasing", {"cu": cu(0, 9, 8), "batch": 2}), ("start at 0", {"cu": cu(1, 8)}),
                       ("x missing", {"x": None}), ("x_stride", {"xs": 63}), ("misaligned", {"x": x.data_ptr() + 2}),
                       ("eps", {"eps": 0.0}), ("y missing", {"y": None})):
        refused(match, "sc_group_norm", *gn(**bad))
    refused("dy or stats", "sc_group_norm_backward", x.data_ptr(), 64, None, None, None, stats.data_ptr(), y.data_ptr(),
            None, None, cu(0, 8), 1, 64, 8, 0, 0, 0)
    q, k, v, lam, _ = _da_inputs(cuda, 8, 8, 2, 1, BF, 57)
    out, offs = torch.empty(8, 2, 128, device=cuda, dtype=BF), cu(0, 8)
    good = dict(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), lam=lam.data_ptr(), q_stride=256, k_stride=128,
                v_stride=128, cu_seqlens_q=ctypes.addressof(offs), cu_seqlens_kv=ctypes.addressof(offs), batch=1,
                heads=2, kv_heads=1, lam_count=2, scale=0.125, dtype=L.SC_BF16, lam_dtype=L.SC_F32, out=out.data_ptr())
    for match, bad in (("bf16 or f16", {"dtype": L.SC_F32}), ("heads", {"heads": 3, "kv_heads": 2}),
                       ("heads", {"heads": 40000}), ("scale", {"scale": 0.0}), ("scale", {"scale": float("nan")}),
                       ("lam_count", {"lam_count": 3}), ("lam must", {"lam_dtype": L.SC_F16}),
                       ("q missing", {"q": None}), ("q missing", {"q": q.data_ptr() + 2}),
                       ("q missing", {"q_stride": 260}), ("k or v", {"k_stride": 120}), ("k or v", {"v": None}),
                       ("out missing", {"out": None}), ("go together", {"lse": stats.data_ptr()})):
        refused(match, "sc_diff_attention", ctypes.byref(L.ScDiffAttentionArgs(**{**good, **bad})))
    refused("backward needs", "sc_diff_attention_backward",
            ctypes.byref(L.ScDiffAttentionArgs(**{**good, "dq": q.data_ptr()})))
    refused("null arguments", "sc_diff_attention", None)
    engine.call("sc_diff_attention", ctypes.byref(L.ScDiffAttentionArgs(**good)))
    assert torch.equal(out, pkg.sparse_diff_attention(q, k, v, lam, [0, 8]))
    engine.call("sc_group_norm", *gn())
    assert torch.equal(y, pkg.sparse_group_norm(x, 8))


# ------------------------------------------------------------------- together
def test_out_is_known_to_autograd(pkg, cuda):
    """A tensor that a backward pass saved may not be overwritten unnoticed; one that requires grad is no out."""
    x, w, b, dy = _gn_inputs(cuda, 40, 64, BF, BF, 14)
    q, k, v, _, _ = _da_inputs(cuda, 40, 40, 1, 1, BF, 67)
    for write in (lambda t: pkg.sparse_group_norm(t, 8, w, b, out=t),
                  lambda t: pkg.sparse_diff_attention(q[:20], k, v, 0.5, [0, 20], [0, 40], out=t.view(20, 1, 128))):
        t, scale = x.clone(), torch.ones((), device=cuda, dtype=BF, requires_grad=True)
        loss = (t * scale).sum()
        write(t)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    out = torch.empty_like(x).requires_grad_()
    with pytest.raises(ValueError, match="requires grad"):
        pkg.sparse_group_norm(x, 8, w, b, out=out)
    with torch.no_grad():
        assert pkg.sparse_group_norm(x, 8, w, b, out=out) is out
    with torch.inference_mode():
        t = x.clone()
        assert torch.equal(pkg.sparse_group_norm(t, 8, w, b, out=t), out)


def test_forward_mode_is_refused(pkg, cuda):
    """No tangent is dropped: torch's own error names the missing rule."""
    from torch.autograd import forward_ad
    x, w, b, dy = _gn_inputs(cuda, 40, 64, FP, FP, 13)
    q, k, v, lam, _ = _da_inputs(cuda, 40, 40, 2, 1, BF, 66)
    with forward_ad.dual_level():
        for call in (lambda: pkg.sparse_group_norm(forward_ad.make_dual(x, dy), 8, w, b),
                     lambda: pkg.sparse_group_norm(x, 8, forward_ad.make_dual(w, b), b),
                     lambda: pkg.sparse_diff_attention(forward_ad.make_dual(q, q.clone()), k, v, lam, [0, 40]),
                     lambda: pkg.sparse_diff_attention(q, k, v, forward_ad.make_dual(lam, lam.clone()), [0, 40])):
            with pytest.raises((RuntimeError, NotImplementedError)):
                call()
            with torch.no_grad(), pytest.raises((RuntimeError, NotImplementedError)):
                call()
        assert pkg.sparse_group_norm(x, 8, w, b).shape == x.shape
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(lambda t: pkg.sparse_group_norm(t, 8, w, b), (x,), (dy,))


def _block(pkg, x, p, cu, heads, kv_heads):
    """Norm, fused projection, differential attention, projection, skip."""
    y = pkg.sparse_group_norm(x, 32, p["w"], p["b"], cu_seqlens=cu, silu=True)
    f = y @ p["qkv"]
    nq, nk = 128 * heads, 128 * kv_heads
    q = f[:, :nq].unflatten(1, (2 * heads, 64))
    k = f[:, nq:nq + nk].unflatten(1, (2 * kv_heads, 64))
    v = f[:, nq + nk:].unflatten(1, (kv_heads, 128))
    return x + pkg.sparse_diff_attention(q, k, v, p["lam"], cu).flatten(1) @ p["o"]


def _block_inputs(cuda, n, c, heads, kv_heads, seed):
    rng = np.random.default_rng(seed)
    mk = lambda s, *shape: torch.from_numpy((s * rng.standard_normal(shape)).astype(np.float32)).to(cuda, BF)  # noqa: E731
    p = {"w": 1 + mk(0.2, c), "b": mk(0.2, c), "qkv": mk(2 * c ** -0.5, c, 128 * (heads + 2 * kv_heads)),
         "o": mk((128 * heads) ** -0.5, 128 * heads, c), "lam": mk(0.1, heads) + 0.5}
    return mk(1.0, n, c), p, mk(1.0, n, c)


def test_block_of_both(pkg, cuda):
    """The two operators in the block they form, values and gradients against
    float64 autograd of the same formulas: about eight roundings to bf16 in a
    row, each below u of a term that reaches the result unscaled."""
    cu, c, heads, kv_heads = [0, 260, 261, 700], 128, 4, 2
    x, p, dy = _block_inputs(cuda, 700, c, heads, kv_heads, 40)
    leaves = [t.requires_grad_() for t in (x, *p.values())]
    y = _block(pkg, x, p, cu, heads, kv_heads)
    got = [y, *torch.autograd.grad(y, leaves, dy)]

    class Plain:
        @staticmethod
        def sparse_group_norm(x, groups, w, b, cu_seqlens, silu):
            parts = []
            for lo, hi in zip(cu_seqlens, cu_seqlens[1:]):
                t = x[lo:hi].reshape(hi - lo, groups, -1)
                m = t.mean((0, 2), keepdim=True)
                parts.append(((t - m) / (t.var((0, 2), unbiased=False, keepdim=True) + 1e-5).sqrt()).flatten(1))
            z = torch.cat(parts) * w + b
            return z * torch.sigmoid(z)

        @staticmethod
        def sparse_diff_attention(q, k, v, lam, cu):
            rows = []
            for lo, hi in zip(cu, cu[1:]):
                hs = []
                for h in range(heads):
                    g = h // (heads // kv_heads)
                    a = [torch.softmax(q[lo:hi, 2 * h + m] @ k[lo:hi, 2 * g + m].T / 8, -1) for m in (0, 1)]
                    hs.append((a[0] - lam[h] * a[1]) @ v[lo:hi, g])
                rows.append(torch.stack(hs, 1))
            return torch.cat(rows)
    x64, p64 = x.detach().double().requires_grad_(), {n: t.detach().double().requires_grad_() for n, t in p.items()}
    y64 = _block(Plain, x64, p64, cu, heads, kv_heads)
    ref = [y64, *torch.autograd.grad(y64, [x64, *p64.values()], dy.double())]
    for name, a, b in zip(("y", "x", *p), got, ref):
        assert _rel(_f64(a), _f64(b)) < 8 * _half(BF), (name, _rel(_f64(a), _f64(b)))


def test_repeatable_and_on_other_streams(pkg, cuda):
    x, p, dy = _block_inputs(cuda, 900, 128, 4, 2, 41)
    leaves = [t.requires_grad_() for t in (x, *p.values())]

    def run():
        y = _block(pkg, x, p, [0, 300, 900], 4, 2)
        return [y, *torch.autograd.grad(y, leaves, dy)]
    ref = run()
    assert all(torch.equal(a, b) for a, b in zip(run(), ref))
    streams = [torch.cuda.Stream(cuda) for _ in range(3)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream(cuda))
        with torch.cuda.stream(s):
            got.append(run())
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, ref))
    pkg.get_engine(cuda).synchronize()


def test_synchronize_waits_for_every_stream(pkg, cuda):
    """Work that was called for on other streams than the last one, and in a replayed graph, is over after it."""
    engine, x = pkg.get_engine(cuda), torch.randn(300, 64, device=cuda)
    side, graph = torch.cuda.Stream(cuda), torch.cuda.CUDAGraph()
    pkg.sparse_group_norm(x, 8)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        pkg.sparse_group_norm(x, 8)
    for replay in (False, True):
        with torch.cuda.stream(side):
            torch.cuda._sleep(200_000_000)  # about 0.1 s
            graph.replay() if replay else pkg.sparse_group_norm(x, 8)
        pkg.sparse_group_norm(x, 8)
        assert not side.query()
        engine.synchronize()
        assert side.query()


def test_from_several_threads(pkg, cuda):
    import threading
    x, p, dy = _block_inputs(cuda, 500, 128, 4, 2, 42)
    leaves = [t.requires_grad_() for t in (x, *p.values())]

    def run():
        y = _block(pkg, x, p, [0, 500], 4, 2)
        return [y, *torch.autograd.grad(y, leaves, dy)]
    ref, bad = run(), []
    torch.cuda.synchronize()

    def work():
        with torch.cuda.stream(torch.cuda.Stream(cuda)):
            for _ in range(10):
                g = run()
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(g, ref)):
                    bad.append(1)
    ts = [threading.Thread(target=work) for _ in range(4)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not bad


def test_group_norm_from_two_handles(pkg, cuda):
    """Calls of one kernel with more and with less shared memory at the same time, a handle per thread."""
    import ctypes
    import threading
    x = torch.randn(2, 4096, device=cuda, dtype=BF)
    cu = (ctypes.c_int32 * 2)(0, 2)
    bad = []

    def work(groups, stream):
        engine, y = pkg.Engine(cuda), torch.empty_like(x)
        with torch.cuda.stream(stream):
            ref = pkg.sparse_group_norm(x, groups)
            try:
                for _ in range(4000):
                    engine.call("sc_group_norm", x.data_ptr(), 4096, None, None, y.data_ptr(), None, cu, 1, 4096,
                                groups, 1e-5, 0, pkg._lib.SC_BF16, pkg._lib.SC_BF16)
                stream.synchronize()
                if not torch.equal(y, ref):
                    bad.append("values")
            except Exception as e:  # noqa: BLE001
                bad.append(e)
        engine.close()
    torch.cuda.synchronize()
    ts = [threading.Thread(target=work, args=(g, torch.cuda.Stream(cuda))) for g in (4096, 2048, 4096, 2048)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not bad, bad


def test_captured_and_replayed(pkg, cuda):
    """Forward and backward of the block in a CUDA graph, two graphs replayed
    in turn with new inputs, against eager calls."""
    cu = [0, 40, 41, 300]
    graphs = []
    for seed in (43, 44):
        x, p, dy = _block_inputs(cuda, 300, 128, 4, 2, seed)
        leaves = [t.requires_grad_() for t in (x, *p.values())]

        def run(x=x, p=p, dy=dy, leaves=leaves):
            y = _block(pkg, x, p, cu, 4, 2)
            return [y.detach(), *torch.autograd.grad(y, leaves, dy)]
        s = torch.cuda.Stream(cuda)
        s.wait_stream(torch.cuda.current_stream(cuda))
        with torch.cuda.stream(s):
            run()
        torch.cuda.current_stream(cuda).wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = run()
        graphs.append((g, got, run, x, dy))
    for k in range(3):
        for g, got, run, x, dy in graphs:
            with torch.no_grad():
                x.copy_(torch.randn_like(x))
                dy.copy_(torch.randn_like(dy))
            g.replay()
            held = [t.clone() for t in got]
            assert all(torch.equal(a, b) for a, b in zip(held, run()))


def test_captured_with_many_sequences(pkg, cuda):
    """A table too long for kernel parameters is written by kernels, so it is captured too."""
    lens = np.random.default_rng(45).integers(0, 5, 300).tolist()
    cu = _cu(lens)
    q, k, v, lam, _ = _da_inputs(cuda, cu[-1], cu[-1], 2, 2, BF, 46)
    x, w, b, _ = _gn_inputs(cuda, cu[-1], 64, BF, BF, 47)

    def run():
        return (pkg.sparse_diff_attention(q, k, v, lam, cu, causal=True),
                pkg.sparse_group_norm(x, 8, w, b, cu_seqlens=cu))
    run()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = run()
    q.copy_(torch.randn_like(q))
    x.copy_(torch.randn_like(x))
    g.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, run()))
