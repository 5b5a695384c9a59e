"""Group norm over sparse sequences and varlen differential attention: cases, plain forms and calls.

Two operators of an attention block over voxels (or tokens): the group norm
that feeds it and the differential attention itself.

* ``gn``: rows ``x`` (N, C) of sequences concatenated along the rows, channels
  last, C in G groups.  Each (sequence, group) is normalised with its own mean
  and variance over rows and channels, then weight, bias and optionally SiLU.
* ``attn``: q (N, 2H, 64), k (N_kv, 2H_kv, 64), v (N_kv, H_kv, 128), lam (H,).
  Head h reads key / value head g = h // (H / H_kv):
  ``out_h = (softmax(c q_2h k_2g^T) - lam_h softmax(c q_2h+1 k_2g+1^T)) v_g``
  inside each sequence, c = 1/8; with "causal" query i of a sequence sees the
  keys j <= i + len_kv - len_q.  A row that sees no key is zero.

"train" adds the gradients of every input.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

EPS = 1e-5
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # one small object in a batch of two: a call whose time is its launches
        {"name": "gn_small", "op": "gn", "lens": "77,129", "c": 64, "groups": 32, "dtype": "bf16", "wdtype": "bf16",
         "silu": True, "train": False},
        # the 64^3 shell's voxels in f32, a training step
        {"name": "gn_shell_f32_train", "op": "gn", "lens": "15068", "c": 64, "groups": 32, "dtype": "f32",
         "wdtype": "f32", "silu": True, "train": True},
        # the ResBlock batch (four shapes at 128^3, 256 channels), a training step with f32 weights
        {"name": "gn_resblock_train", "op": "gn", "lens": "30211,33817,41002,28694", "c": 256, "groups": 32,
         "dtype": "bf16", "wdtype": "f32", "silu": True, "train": True},
        # the 256^3 union of shells at 128 channels
        {"name": "gn_shells", "op": "gn", "lens": "406351", "c": 128, "groups": 32, "dtype": "bf16",
         "wdtype": "bf16", "silu": True, "train": False},
        # rows that are no whole number of 16-byte words, ragged sequences, one of a row and one of none
        {"name": "gn_odd_f16_train", "op": "gn", "lens": "5003,1,0,12011,257", "c": 36, "groups": 9, "dtype": "f16",
         "wdtype": "f16", "silu": False, "train": True},
        # one token of one sequence against a short cache: latency
        {"name": "attn_step_small", "op": "attn", "lens_q": "1", "lens_kv": "300", "heads": 8, "kv_heads": 8,
         "dtype": "f16", "causal": False, "train": False},
        # one token of each of 24 sequences against ragged caches, shared key heads
        {"name": "attn_step_batch", "op": "attn", "lens_q": ",".join(["1"] * 24),
         "lens_kv": ",".join(str(513 + 677 * i) for i in range(24)), "heads": 16, "kv_heads": 4, "dtype": "bf16",
         "causal": True, "train": False},
        # the two objects of the attention benchmark, forward (sampling)
        {"name": "attn_objects", "op": "attn", "lens_q": "10000,6384", "lens_kv": "10000,6384", "heads": 8,
         "kv_heads": 8, "dtype": "bf16", "causal": False, "train": False},
        # a training step on two objects
        {"name": "attn_objects_train", "op": "attn", "lens_q": "8192,2777", "lens_kv": "8192,2777", "heads": 8,
         "kv_heads": 8, "dtype": "bf16", "causal": False, "train": True},
        # cross attention on ragged pairs, one without keys and one without queries, shared key heads
        {"name": "attn_cross_odd_train", "op": "attn", "lens_q": "70,0,200,33,1029", "lens_kv": "130,9,1,0,777",
         "heads": 6, "kv_heads": 2, "dtype": "f16", "causal": False, "train": True},
        # token sequences, causal, shared key heads, a training step
        {"name": "attn_causal_train", "op": "attn", "lens_q": "2048,1023,300", "lens_kv": "2048,1023,300",
         "heads": 16, "kv_heads": 4, "dtype": "bf16", "causal": True, "train": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.45:
        groups = rng.choice([1, 4, 8, 9, 16, 32])
        c = groups * rng.randint(max(1, 24 // groups), max(2, 320 // groups))
        total = _log(rng, 64, max(64, min(400000, 24000000 // c)))
        n = rng.randint(1, 5)
        cuts = [rng.uniform(0.6, 1.4) for _ in range(n)]
        lens = [max(1, int(total * w / sum(cuts))) for w in cuts]
        if rng.random() < 0.2:
            lens.append(rng.choice([0, 1]))
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        return {"op": "gn", "lens": ",".join(map(str, lens)), "c": c, "groups": groups, "dtype": dtype,
                "wdtype": rng.choice([dtype, "f32"]), "silu": rng.random() < 0.6, "train": rng.random() < 0.5}
    dtype, kv_heads = rng.choice(["bf16", "bf16", "f16"]), rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4] if kv_heads < 8 else [1, 2])
    if rng.random() < 0.4:  # single tokens against a cache
        n = _log(rng, 1, 40)
        top = max(64, min(16000, 200000 // n))
        kv = [rng.randint(max(1, top // 8), top) for _ in range(n)]
        return {"op": "attn", "lens_q": ",".join(["1"] * n), "lens_kv": ",".join(map(str, kv)), "heads": heads,
                "kv_heads": kv_heads, "dtype": dtype, "causal": rng.random() < 0.5, "train": False}
    train, causal = rng.random() < 0.6, rng.random() < 0.4
    n = rng.randint(1, 4)
    top = _log(rng, 32, 6000 if n == 1 else 3500)
    q = [rng.randint(max(1, top // 2), top) for _ in range(n)]
    kv = q if causal or rng.random() < 0.6 else [rng.randint(max(1, top // 2), top) for _ in range(n)]
    return {"op": "attn", "lens_q": ",".join(map(str, q)), "lens_kv": ",".join(map(str, kv)), "heads": heads,
            "kv_heads": kv_heads, "dtype": dtype, "causal": causal, "train": train}


def _lens(text):
    return [int(t) for t in text.split(",")]


def _offsets(text):
    cu = [0]
    for n in _lens(text):
        cu.append(cu[-1] + n)
    return cu


def _package():
    """The framework's package (its folder's name is no identifier), as a user's program loads it."""
    if "sparseconv_b200" not in sys.modules:
        folder = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                              "trellis.2-stableprojectorz_b200")
        spec = importlib.util.spec_from_file_location("sparseconv_b200", os.path.join(folder, "__init__.py"),
                                                      submodule_search_locations=[folder])
        sys.modules["sparseconv_b200"] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules["sparseconv_b200"])
    return sys.modules["sparseconv_b200"]


def prepare(case, seed):
    dt = DTYPES[case["dtype"]]
    gen = torch.Generator("cuda").manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    state = dict(case)
    if case["op"] == "gn":
        cu, c = _offsets(case["lens"]), case["c"]
        wt = DTYPES[case["wdtype"]]
        # activations: channels with offsets and scales of their own
        x = normal(cu[-1], c) * (0.5 + normal(c).abs()) + 0.7 * normal(c)
        state.update(cu=cu, x=x.to(dt), w=(1 + 0.2 * normal(c)).to(wt), b=(0.2 * normal(c)).to(wt))
        if case["train"]:
            state["dy"] = normal(cu[-1], c).to(dt)
        leaves = ("x", "w", "b")
    else:
        cu_q, cu_kv = _offsets(case["lens_q"]), _offsets(case["lens_kv"])
        h, hk = case["heads"], case["kv_heads"]
        # scores of deviation 1.5; values with channel means; lambda between 0.2 and 0.8 as layers learn it
        mean = 0.5 * normal(hk, 128)
        state.update(cu_q=cu_q, cu_kv=cu_kv, q=(1.5 * normal(cu_q[-1], 2 * h, 64)).to(dt),
                     k=normal(cu_kv[-1], 2 * hk, 64).to(dt), v=(normal(cu_kv[-1], hk, 128) + mean).to(dt),
                     lam=(0.2 + 0.6 * torch.rand(h, generator=gen, device="cuda")).to(dt))
        if case["train"]:  # leans along the output, as a squared error's gradient does
            state["dout"] = (normal(cu_q[-1], h, 128) + mean.repeat_interleave(h // hk, 0)).to(dt)
        leaves = ("q", "k", "v", "lam")
    if case["train"]:
        for name in leaves:
            state[name].requires_grad_()
    return state


def _rows(cu):
    """Padded view of concatenated rows: their index (B, L), and which of them are there; None for one sequence."""
    if len(cu) == 2:
        return None
    at = torch.tensor(cu, device="cuda")
    i = torch.arange(max(b - a for a, b in zip(cu, cu[1:])), device="cuda")
    there = i[None] < (at[1:] - at[:-1])[:, None]
    return torch.where(there, at[:-1, None] + i[None], 0), there


def _pad(x, rows):
    if rows is None:
        return x[None]
    return x[rows[0]] * rows[1].reshape(rows[1].shape + (1,) * (x.dim() - 1))


def _unpad(x, rows):
    return x[0] if rows is None else x[rows[1]]


def _gn_plain(s):
    dt, wt, g = s["x"].dtype, s["w"].dtype, s["groups"]
    rows = _rows(s["cu"])
    x = _pad(s["x"].detach().float(), rows)  # (B, L, C)
    b, n, c = x.shape
    grouped = lambda t: t.reshape(b, n, g, c // g)  # noqa: E731
    there = 1.0 if rows is None else rows[1][:, :, None, None].float()
    lens = torch.tensor([[hi - lo] for lo, hi in zip(s["cu"], s["cu"][1:])], device="cuda")
    count = (lens.clamp(min=1) * (c // g)).float()  # (B, 1)
    mean = grouped(x).sum((1, 3)) / count
    d = (grouped(x) - mean[:, None, :, None]) * there
    rstd = ((d * d).sum((1, 3)) / count + EPS).rsqrt()
    xhat = (d * rstd[:, None, :, None]).reshape(b, n, c)
    w, bias = s["w"].detach().float(), s["b"].detach().float()
    z = xhat * w + bias
    sig = 1 / (1 + torch.exp(-z)) if s["silu"] else None
    y = _unpad(z * sig if s["silu"] else z, rows).to(dt)
    if not s["train"]:
        return {"y": y}
    dz = _pad(s["dy"].float(), rows)
    if s["silu"]:
        dz = dz * sig * (1 + z * (1 - sig))
    dw, db = (dz * xhat).sum((0, 1)).to(wt), dz.sum((0, 1)).to(wt)
    dx = grouped(dz * w)
    m1 = (dx.sum((1, 3)) / count)[:, None, :, None]
    m2 = ((dx * grouped(xhat)).sum((1, 3)) / count)[:, None, :, None]
    dx = (dx - m1 - grouped(xhat) * m2) * rstd[:, None, :, None]
    return {"y": y, "dx": _unpad(dx.reshape(b, n, c), rows).to(dt), "dw": dw, "db": db}


def _attn_plain(s):
    dt, h, hk = s["q"].dtype, s["heads"], s["kv_heads"]
    r = h // hk
    rq, rk = _rows(s["cu_q"]), _rows(s["cu_kv"])
    q, k, v = (_pad(s[n].detach().float(), rows) for n, rows in (("q", rq), ("k", rk), ("v", rk)))
    b, n, m = q.shape[0], q.shape[1], k.shape[1]
    lam = s["lam"].detach().float().reshape(hk, r, 1, 1)
    q = q.reshape(b, n, hk, r, 2, 64).permute(0, 2, 4, 3, 1, 5).reshape(b, hk, 2, r * n, 64)
    k = k.reshape(b, m, hk, 2, 64).permute(0, 2, 3, 1, 4)  # (B, Hk, 2, M, 64)
    v = v.permute(0, 2, 1, 3)  # (B, Hk, M, 128)
    i, j = torch.arange(n, device="cuda"), torch.arange(m, device="cuda")
    lq = torch.tensor([hi - lo for lo, hi in zip(s["cu_q"], s["cu_q"][1:])], device="cuda")[:, None, None]
    lk = torch.tensor([hi - lo for lo, hi in zip(s["cu_kv"], s["cu_kv"][1:])], device="cuda")[:, None, None]
    see = (j < lk) & (i[:, None] < lq)
    if s["causal"]:
        see = see & (j <= i[:, None] + lk - lq)
    see = see[:, None, None, None]  # (B, 1, 1, 1, N, M)
    score = (q @ k.transpose(-1, -2) * 0.125).reshape(b, hk, 2, r, n, m)
    score = torch.where(see, score, -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(score - top)
    del score
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    o = (p.reshape(b, hk, 2, r * n, m) @ v[:, :, None]).reshape(b, hk, 2, r, n, 128)
    back = lambda t, rows: _unpad(t, rows).to(dt)  # noqa: E731
    out = back((o[:, :, 0] - lam * o[:, :, 1]).permute(0, 3, 1, 2, 4).reshape(b, n, h, 128), rq)
    if not s["train"]:
        return {"out": out}
    do = _pad(s["dout"].float(), rq).reshape(b, n, hk, r, 128).permute(0, 2, 3, 1, 4)  # (B, Hk, r, N, 128)
    dlam = -(do * o[:, :, 1]).sum((0, 3, 4)).reshape(h)
    dp = (do.reshape(b, hk, r * n, 128) @ v.transpose(-1, -2)).reshape(b, hk, r, n, m)
    diff = p[:, :, 0] - lam * p[:, :, 1]
    dv = diff.reshape(b, hk, r * n, m).transpose(-1, -2) @ do.reshape(b, hk, r * n, 128)
    del diff
    sign = torch.stack((torch.ones_like(lam), -lam))[None].transpose(1, 2)  # (1, Hk, 2, r, 1, 1)
    delta = (do[:, :, None] * o).sum(-1, keepdim=True)
    ds = ((p * (dp[:, :, None] - delta)) * (sign * 0.125)).reshape(b, hk, 2, r * n, m)
    del p, dp
    dq = (ds @ k).reshape(b, hk, 2, r, n, 64).permute(0, 4, 1, 3, 2, 5).reshape(b, n, 2 * h, 64)
    dk = (ds.transpose(-1, -2) @ q).permute(0, 3, 1, 2, 4).reshape(b, m, 2 * hk, 64)
    return {"out": out, "dq": back(dq, rq), "dk": back(dk, rk), "dv": back(dv.permute(0, 2, 1, 3), rk),
            "dlam": dlam.to(s["lam"].dtype)}


def run(state):
    s = state
    if not own:
        return _gn_plain(s) if s["op"] == "gn" else _attn_plain(s)
    pkg = _package()
    if s["op"] == "gn":
        y = pkg.sparse_group_norm(s["x"], s["groups"], s["w"], s["b"], EPS, cu_seqlens=s["cu"], silu=s["silu"])
        if not s["train"]:
            return {"y": y}
        dx, dw, db = torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"])
        return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}
    out = pkg.sparse_diff_attention(s["q"], s["k"], s["v"], s["lam"], s["cu_q"], s["cu_kv"], causal=s["causal"])
    if not s["train"]:
        return {"out": out}
    dq, dk, dv, dlam = torch.autograd.grad(out, (s["q"], s["k"], s["v"], s["lam"]), s["dout"])
    return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv, "dlam": dlam}


def _pairs(case):
    """(query, key) pairs of one head that the mask leaves."""
    total = 0
    for n, m in zip(_lens(case["lens_q"]), _lens(case["lens_kv"])):
        if case["causal"]:  # row i of n sees min(m, max(0, i + 1 + m - n)) keys
            lo = max(0, n - m)
            first = max(0, m - n) + 1 if n > lo else 0
            total += (n - lo) * (first + m) // 2
        else:
            total += n * m
    return total


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "gn":
        n, c = sum(_lens(case["lens"])), case["c"]
        wsize = 4 if case["wdtype"] == "f32" else 2
        # forward: x read, y written; training: dy read and dx written besides
        return {"bytes": n * c * size * (4 if case["train"] else 2) + c * wsize * (4 if case["train"] else 2),
                "flops": n * c * (20 if case["train"] else 8)}
    h, hk = case["heads"], case["kv_heads"]
    nq, nkv = sum(_lens(case["lens_q"])), sum(_lens(case["lens_kv"]))
    qo, kv = nq * h * 256 * size, nkv * hk * 256 * size  # q and out; k and v
    bytes_, flops = qo + kv, 768 * _pairs(case) * h
    if case["train"]:  # dout read, dq, dk and dv written; scores again, dp, dv, dq and dk
        bytes_ += qo + kv
        flops += 1280 * _pairs(case) * h
    return {"bytes": bytes_, "flops": flops}


def _gn_exact(s):
    x, w, b = (s[n].detach().double().requires_grad_(s["train"]) for n in ("x", "w", "b"))
    parts = []
    for lo, hi in zip(s["cu"], s["cu"][1:]):
        if hi == lo:
            continue
        part = x[lo:hi].reshape(hi - lo, s["groups"], -1)
        var, mean = torch.var_mean(part, (0, 2), unbiased=False, keepdim=True)
        parts.append(((part - mean) / torch.sqrt(var + EPS)).reshape(hi - lo, -1))
    y = torch.cat(parts) * w + b
    if s["silu"]:
        y = y * torch.sigmoid(y)
    if not s["train"]:
        return {"y": y}
    dx, dw, db = torch.autograd.grad(y, (x, w, b), s["dy"].double())
    return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}


def _attn_exact(s):
    q, k, v, lam = (s[n].detach().double() for n in ("q", "k", "v", "lam"))
    h, hk, train = s["heads"], s["kv_heads"], s["train"]
    out = torch.zeros(q.shape[0], h, 128, dtype=torch.float64, device="cuda")
    dq, dk, dv, dlam = (torch.zeros_like(t) for t in (q, k, v, lam))
    for (q0, q1, k0, k1) in zip(s["cu_q"], s["cu_q"][1:], s["cu_kv"], s["cu_kv"][1:]):
        if q1 == q0 or k1 == k0:
            continue
        for head in range(h):
            g = head // (h // hk)
            kk, vv, ll = k[k0:k1, 2 * g:2 * g + 2].clone(), v[k0:k1, g].clone(), lam[head].clone()
            for lo in range(q0, q1, 4096):  # queries are independent of one another
                hi = min(q1, lo + 4096)
                qq = q[lo:hi, 2 * head:2 * head + 2].clone()
                given = [t.detach().requires_grad_(train) for t in (qq, kk, vv, ll)]
                maps, dead = [], None
                for one in (0, 1):
                    a = given[0][:, one] @ given[1][:, one].T / 8
                    if s["causal"]:
                        i = torch.arange(lo - q0, hi - q0, device="cuda")[:, None]
                        hidden = torch.arange(k1 - k0, device="cuda")[None] > i + (k1 - k0) - (q1 - q0)
                        dead = hidden.all(1, keepdim=True)
                        a = a.masked_fill(hidden & ~dead, -math.inf)
                    a = torch.softmax(a, -1)
                    maps.append(a if dead is None else a.masked_fill(dead, 0.0))
                o = (maps[0] - given[3] * maps[1]) @ given[2]
                out[lo:hi, head] = o.detach()
                if train:
                    got = torch.autograd.grad(o, given, s["dout"][lo:hi, head].double())
                    dq[lo:hi, 2 * head:2 * head + 2] = got[0]
                    dk[k0:k1, 2 * g:2 * g + 2] += got[1]
                    dv[k0:k1, g] += got[2]
                    dlam[head] += got[3]
    return {"out": out, "dq": dq, "dk": dk, "dv": dv, "dlam": dlam} if train else {"out": out}


def exact(case, seed):
    s = prepare(case, seed)
    return _gn_exact(s) if s["op"] == "gn" else _attn_exact(s)
