"""The training operators around the stone attention: ``fused_attention_relative``,
``policy_log_probs`` and ``residual_dropout``.

CPU: registration, argument checks, fake shapes, the bucket table and the
generator's reference.  GPU: values and gradients against float64 statements
of the formulas on the CPU.  A tolerance is a sum of what the kernel rounds:
half a step of the output's type relative to the value, and fp32 (or, where
noted, 16-bit) errors relative to the sum of the absolute terms that the
value is made of, computed beside it.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import mantisnet  # noqa: F401  registers the operators
from mantisnet import ops, tables

OPS = torch.ops.mantisnet
INF = math.inf
HALF_STEP = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
gpu = pytest.mark.gpu


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _within(got, exp, tol, what):
    """|got - exp| <= tol elementwise; infinities and NaNs exactly where expected."""
    got, exp, tol = got.detach().cpu().double(), exp.double(), torch.as_tensor(tol).double().expand(exp.shape)
    assert got.shape == exp.shape, what
    assert torch.equal(got.isnan(), exp.isnan()), what
    fin = exp.isfinite()
    assert torch.equal(got[~fin & ~exp.isnan()], exp[~fin & ~exp.isnan()]), what
    over = (got[fin] - exp[fin]).abs() - tol[fin]
    assert over.numel() == 0 or float(over.max()) <= 0, (what, float(over.max()), float(exp[fin].abs().max()))


# ----------------------------------------------------------------- the formulas in float64


def _pairs(coords, buckets, n, n_latents, n_buckets):
    """(n, n) bucket of each (query, key) of one position; -1 where the table's entry is no bucket."""
    hq, hr = (buckets.shape[0] - 1) // 2, (buckets.shape[1] - 1) // 2
    c = coords[:n].long()
    d = c[None] - c[:, None]
    pair = buckets.long()[d[..., 0].clamp(-hq, hq) + hq, d[..., 1].clamp(-hr, hr) + hr]
    pair = torch.where((pair < 0) | (pair >= n_buckets), -1, pair)
    pair[:n_latents] = n_buckets - 1
    pair[:, :n_latents] = n_buckets - 2
    return pair


def relative_reference(q, k, v, bias, coords, buckets, seq_lens, n_latents, grad=None):
    """Values, gradients and, for each, the sum of absolute terms (``amp``) in float64."""
    q, k, v, bias = (x.detach().cpu().double() for x in (q, k, v, bias))
    coords, buckets, seq_lens = coords.cpu(), buckets.cpu(), seq_lens.cpu()
    grad = None if grad is None else grad.detach().cpu().double()
    p, a, t, d = q.shape
    val = {n: torch.zeros_like(q) for n in ("out", "dq", "dk", "dv")}
    val.update(lse=q.new_zeros(p, a, t), dbias=torch.zeros_like(bias))
    amp = {n: torch.zeros_like(x) for n, x in val.items()}
    score = 0.0
    for i in range(p):
        n = min(max(int(seq_lens[i]), 0), t)
        if n == 0:
            continue
        pair = _pairs(coords[i], buckets, n, n_latents, bias.shape[1])
        known = pair >= 0
        for h in range(a):
            qq, kk, vv = q[i, h, :n], k[i, h, :n], v[i, h, :n]
            b = torch.where(known, bias[h][pair.clamp(min=0)], 0.0)
            s = qq @ kk.T / math.sqrt(d) + b
            finite = torch.where(b.isfinite() & (b.abs() < 1e30), b.abs(), 0.0)
            score = max(score, float((qq.abs() @ kk.abs().T / math.sqrt(d) + finite).max()))
            m = s.amax(1, keepdim=True)
            m = torch.where(m == -INF, 0.0, m)
            e = torch.exp(s - m)
            z = e.sum(1, keepdim=True)
            pr = torch.where(z == 0, 0.0, e / z)
            val["out"][i, h, :n], amp["out"][i, h, :n] = pr @ vv, pr @ vv.abs()
            val["lse"][i, h, :n] = (m + torch.log(z))[:, 0]
            if grad is None:
                continue
            go = grad[i, h, :n]
            dp, dpa = go @ vv.T, go.abs() @ vv.abs().T
            ds = pr * (dp - (pr * dp).sum(1, keepdim=True))
            dsa = pr * (dpa + (pr * dpa).sum(1, keepdim=True))
            r = 1 / math.sqrt(d)
            for name, x, xa in (("dq", ds @ kk * r, dsa @ kk.abs() * r), ("dk", ds.T @ qq * r, dsa.T @ qq.abs() * r),
                                ("dv", pr.T @ go, pr.T @ go.abs())):
                val[name][i, h, :n], amp[name][i, h, :n] = x, xa
            val["dbias"][h].index_add_(0, pair[known], ds[known])
            amp["dbias"][h].index_add_(0, pair[known], dsa[known])
    return val, amp, score


def _relative_tolerances(val, amp, score, dtype, t, d, parts):
    """fp32: a score of d products and a bias is off by (d + 8) half steps of
    its absolute terms, which is a probability's relative error; a sum of n
    terms adds n half steps.  16-bit: the probabilities of the forward's value
    product are rounded (and so is their sum); the backward's operands keep 16
    bits; outputs round once."""
    u = HALF_STEP[dtype]
    rel = 2 * 2.0**-24 * ((d + 8) * (score + 1) + t + d + 16)
    tiny = 2.0**-25 if dtype == torch.float16 else 0.0  # half a step of the subnormal range
    tol = {n: u * val[n].abs() + (3 * rel + 2.0**-16) * amp[n] * (1 + u) + tiny for n in ("dq", "dk", "dv")}
    # (a probability up to 2^8 under fp16's least step, each of t keys)
    tol["out"] = u * val["out"].abs() + (2 * u + 2 * rel) * amp["out"] * (1 + u) + tiny
    if dtype == torch.float16:
        tol["out"] = tol["out"] + 2.0**-24 * t * float(amp["out"].max())
    fin = torch.where(val["lse"].isfinite(), val["lse"].abs(), 0.0)
    tol["lse"] = rel + 2.0**-23 * (fin + 1)
    tol["dbias"] = (3 * rel + 2.0**-24 * (t + 64 * 4 + parts / 256 + 16)) * amp["dbias"]
    return tol


def relative_case(lens, heads, d, dtype, seed, *, n_latents=4, table=(7, 7), n_buckets=12, spread=3.0, extra=0,
                  device="cpu"):
    g = _gen(seed)
    p, t = len(lens), max(max(lens), 1) + extra
    # rows of a (P, T, A, D) projection
    q, k, v, grad = (torch.randn(p, t, heads, d, generator=g).to(dtype).to(device).transpose(1, 2) for _ in range(4))
    bias = torch.randn(heads, n_buckets, generator=g).to(device)
    coords = (torch.randn(p, t, 2, generator=g) * spread).round().to(torch.int32).to(device)
    buckets = torch.randint(0, n_buckets, table, generator=g).to(torch.int32).to(device)
    return q, k, v, bias, coords, buckets, torch.tensor(lens, dtype=torch.int32, device=device), \
        min(n_latents, t), grad


def _run_relative(case):
    q, k, v, bias, coords, buckets, lens, n_latents, grad = case
    leaves = [x.detach().clone(memory_format=torch.preserve_format).requires_grad_(True) for x in (q, k, v, bias)]
    out, lse, _stats = OPS.fused_attention_relative(*leaves, coords, buckets, lens, n_latents)
    dq, dk, dv, dbias = torch.autograd.grad(out, leaves, grad)
    return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv, "dbias": dbias}


def check_relative(case):
    got = _run_relative(case)
    q, k, v, bias, coords, buckets, lens, n_latents, grad = case
    val, amp, score = relative_reference(q, k, v, bias, coords, buckets, lens, n_latents, grad)
    p, _a, t, d = q.shape
    tol = _relative_tolerances(val, amp, score, q.dtype, t, d, p * (t // 64 + 1))
    for name in got:
        assert got[name].dtype == (q.dtype if name in ("out", "dq", "dk", "dv") else torch.float32), name
        _within(got[name], val[name], tol[name], name)
    return got


def policy_reference(logits, offsets, moves, top, grads=None):
    """Values, the logits' gradient and absolute terms in float64."""
    x, offsets, moves = logits.detach().cpu().double(), offsets.cpu().tolist(), moves.cpu()
    p, g = moves.shape
    val = {"log_probs": torch.zeros(p, g), "entropy": torch.zeros(p), "lse": torch.full((p,), -INF),
           "top_log_probs": torch.full((p, top), -INF), "top_moves": torch.full((p, top), -1)}
    val = {n: t if n == "top_moves" else t.double() for n, t in val.items()}
    dx, amp = torch.zeros_like(x), torch.zeros_like(x)
    err = torch.zeros(p, dtype=torch.float64)  # a log probability's terms
    for i in range(p):
        run = x[offsets[i]:offsets[i + 1]]
        inside = (moves[i] >= 0) & (moves[i] < run.numel())
        if run.isnan().any() or (run == INF).any():
            for n in ("entropy", "lse", "top_log_probs"):
                val[n][i] = math.nan
            val["log_probs"][i][inside] = math.nan
            dx[offsets[i]:offsets[i + 1]] = math.nan
            continue
        if run.numel() == 0 or (run == -INF).all():
            val["log_probs"][i][inside] = -INF
            continue
        above = run - run.max()  # (apart from the maximum: at 1e38 float64 holds no log beside it)
        logp = above - above.exp().sum().log()
        lse = run.max() + above.exp().sum().log()
        pr = logp.exp()
        plogp = torch.where(pr > 0, pr * logp, 0.0)
        order = torch.sort(run, descending=True, stable=True).indices
        order = order[run[order] > -INF][:top]
        val["lse"][i], val["entropy"][i] = lse, -plogp.sum()
        val["log_probs"][i][inside] = logp[moves[i][inside]]
        val["top_moves"][i, :len(order)], val["top_log_probs"][i, :len(order)] = order, logp[order]
        seen = logp[logp > -1e30]
        err[i] = float(seen.abs().max())
        if grads is not None:
            gl, ge, gs, gt = (None if y is None else y.detach().cpu().double() for y in grads)
            common, acc = torch.zeros(()).double(), torch.zeros(()).double()
            at = torch.zeros_like(run)
            at_abs = torch.zeros_like(run)
            if gs is not None:
                common, acc = common + gs[i], acc + gs[i].abs()
            for y, idx in ((gl, moves[i]), (gt, val["top_moves"][i])):
                if y is None:
                    continue
                ok = (idx >= 0) & (idx < run.numel())
                common, acc = common - y[i][ok].sum(), acc + y[i][ok].abs().sum()
                at.index_add_(0, idx[ok], y[i][ok])
                at_abs.index_add_(0, idx[ok], y[i][ok].abs())
            h = val["entropy"][i]
            e = ge[i] if ge is not None else 0.0 * h
            inner = torch.where(pr > 0, logp + h, 0.0)
            dx[offsets[i]:offsets[i + 1]] = pr * (common - e * inner) + at
            amp[offsets[i]:offsets[i + 1]] = pr * (acc + e.abs() * (torch.where(pr > 0, logp.abs(), 0.0) + h)) + at_abs
    return val, dx, amp, err


def check_policy(logits, offsets, moves, top, grads, need_error=False):
    leaf = logits.detach()
    if not leaf.is_contiguous():  # keep the stride
        base = torch.zeros(leaf.numel() * leaf.stride(0), dtype=leaf.dtype, device=leaf.device)
        view = base[::leaf.stride(0)]
        view.copy_(leaf)
        leaf = view
    leaf = leaf.requires_grad_(True)
    out = OPS.policy_log_probs(leaf, offsets, moves, top)
    (dx,) = torch.autograd.grad([o for o, g in zip(out[:4], grads) if g is not None],
                                leaf, [g for g in grads if g is not None])
    if need_error:
        with pytest.raises(ValueError, match="out of range"):
            ops.raise_on_device_error(logits.device)
    else:
        ops.raise_on_device_error(logits.device)
    val, edx, amp, err = policy_reference(logits, offsets, moves, top, grads)
    lens = (offsets[1:] - offsets[:-1]).cpu().double()
    # fp32: a lane's chain of sums, an exponential's argument and value, the log;
    # a log probability's own terms
    rel = 2.0**-23 * (lens / 256 + 48)
    got = dict(zip(("log_probs", "entropy", "lse", "top_log_probs", "top_moves"), out))
    assert torch.equal(got["top_moves"].cpu(), val["top_moves"])
    fin = lambda x: torch.where(x.isfinite(), x.abs(), 0.0)  # noqa: E731
    _within(got["lse"], val["lse"], rel + 2.0**-23 * fin(val["lse"]), "lse")
    _within(got["entropy"], val["entropy"], rel * (2 + err) * 2, "entropy")
    for name in ("log_probs", "top_log_probs"):
        _within(got[name], val[name], (rel + 2.0**-23 * (1 + 2 * err))[:, None] + 2.0**-23 * fin(val[name]), name)
    row = torch.repeat_interleave((rel + 2.0**-22 * (1 + err)) * 4, lens.long())
    covered = torch.zeros_like(edx)
    covered[int(offsets[0]):int(offsets[-1])] = row
    u = HALF_STEP[logits.dtype]
    tiny = 2.0**-25 if logits.dtype == torch.float16 else 2.0**-126
    _within(dx, edx, u * fin(edx) + covered * amp * (1 + u) + tiny, "dlogits")
    assert dx.dtype == logits.dtype and dx.is_contiguous()
    return out, dx


def philox_words(n, seed, step, salt):
    """The first n words (Salmon et al. 2011, Philox4x32-10), in Python integers."""
    mask, out = (1 << 32) - 1, []
    for group in range((n + 3) // 4):
        c = [group & mask, group >> 32, step & mask, salt]
        k = [seed & mask, (seed >> 32) & mask]
        for _ in range(10):
            a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
            c = [(b >> 32) ^ c[1] ^ k[0], b & mask, (a >> 32) ^ c[3] ^ k[1], a & mask]
            k = [(k[0] + 0x9E3779B9) & mask, (k[1] + 0xBB67AE85) & mask]
        out += c
    return np.array(out[:n], dtype=np.uint64)


# ----------------------------------------------------------------- CPU


NAMES = {"fused_attention_relative": 3, "fused_attention_relative_backward": 4, "policy_log_probs": 6,
         "policy_log_probs_backward": 1, "residual_dropout": 1, "residual_dropout_backward": 1}


@pytest.mark.parametrize("name", sorted(NAMES))
def test_registered(name):
    assert len(getattr(OPS, name).default._schema.returns) == NAMES[name]
    assert name in mantisnet.library.OPERATORS


def test_generator_reference_is_the_published_one():
    # the published known answer for a counter and key of zeros
    assert [hex(int(w)) for w in philox_words(4, 0, 0, 0)] == ["0x6627e8d5", "0xe169c58d", "0xbc57ac4c", "0x9b00dbd8"]


@pytest.mark.parametrize("reach", [1, 3, 12, 30])
def test_relative_buckets(reach):
    table, count = tables.relative_buckets(reach)
    assert table.shape == (2 * reach + 3, 2 * reach + 3) and table.dtype == torch.int32 and count == 2 * reach + 4
    assert table.numel() <= 4096
    mid = reach + 1
    for dq in range(-reach - 1, reach + 2):
        for dr in range(-reach - 1, reach + 2):
            dist = (abs(dq) + abs(dr) + abs(dq + dr)) // 2
            axis = 0 in (dq, dr, dq + dr)
            want = 2 * reach + 1 if dist > reach else dist if axis else reach + dist
            assert int(table[mid + dq, mid + dr]) == want
    for bad in (0, 31):
        with pytest.raises(ValueError):
            tables.relative_buckets(bad)


def test_cpu_tensors_are_refused():
    case = relative_case([5, 9], 2, 16, torch.bfloat16, 0)
    with pytest.raises(RuntimeError, match="no CPU path"):
        OPS.fused_attention_relative(*case[:8])
    with pytest.raises(RuntimeError, match="no CPU path"):
        OPS.policy_log_probs(torch.zeros(3), torch.tensor([0, 3]), torch.zeros(1, 1, dtype=torch.long), 1)
    with pytest.raises(RuntimeError, match="no CPU path"):
        OPS.residual_dropout(torch.zeros(3), None, torch.zeros(2, dtype=torch.long), 0.5, 0)


def _fake_relative(**change):
    args = {"q": torch.empty(2, 4, 9, 32, dtype=torch.bfloat16, device="cuda"),
            "bias": torch.empty(4, 12, device="cuda"),
            "coords": torch.empty(2, 9, 2, dtype=torch.int32, device="cuda"),
            "buckets": torch.empty(5, 7, dtype=torch.int32, device="cuda"),
            "seq_lens": torch.empty(2, dtype=torch.int32, device="cuda"), "n_latents": 4}
    args["k"] = args["v"] = args["q"]
    args.update(change)
    return [args[n] for n in ("q", "k", "v", "bias", "coords", "buckets", "seq_lens", "n_latents")]


def test_fakes_and_refusals():
    """Shapes of the fakes, and what the argument checks refuse (fake tensors: nothing is launched)."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        new = lambda *shape, dtype=torch.float32: torch.empty(shape, dtype=dtype, device="cuda")  # noqa: E731
        i64 = torch.int64
        out, lse, stats = OPS.fused_attention_relative(*_fake_relative())
        assert out.shape == (2, 4, 9, 32) and lse.shape == (2, 4, 9) and stats.shape == (2, 4, 9, 2)
        res = OPS.policy_log_probs(new(50, dtype=torch.float16), new(4, dtype=i64), new(3, 2, dtype=i64), 5)
        assert [tuple(r.shape) for r in res] == [(3, 2), (3,), (3,), (3, 5), (3, 5), (3, 2)]
        assert res[4].dtype == i64 and all(r.dtype == torch.float32 for r in res[:4])
        assert OPS.residual_dropout(new(3, 5, dtype=torch.bfloat16), new(3, 5), new(2, dtype=i64), 0.1,
                                    0).dtype == torch.float32
        for change in (
                {"q": new(2, 4, 9, 32)}, {"k": new(2, 4, 8, 32, dtype=torch.bfloat16)},
                {"q": new(2, 4, 9, 24, dtype=torch.bfloat16), "k": new(2, 4, 9, 24, dtype=torch.bfloat16),
                 "v": new(2, 4, 9, 24, dtype=torch.bfloat16)},
                {"v": new(2, 4, 9, 32, dtype=torch.float16)}, {"bias": new(3, 12)}, {"bias": new(4, 385)},
                {"bias": new(4, 0)}, {"bias": new(4, 12, dtype=i64)}, {"bias": new(4, 1)},
                {"coords": new(2, 9, 2)}, {"coords": new(2, 8, 2, dtype=torch.int32)},
                {"buckets": new(4, 7, dtype=torch.int32)}, {"buckets": new(5, 7, dtype=i64)},
                {"buckets": new(65, 65, dtype=torch.int32)}, {"seq_lens": new(2, dtype=i64)},
                {"seq_lens": new(3, dtype=torch.int32)}, {"n_latents": -1}, {"n_latents": 10}):
            with pytest.raises(ValueError):
                OPS.fused_attention_relative(*_fake_relative(**change))
        good = (new(50), new(4, dtype=i64), new(3, 2, dtype=i64), 5)
        for at, bad in ((0, new(50, 1)), (0, new(50, dtype=torch.float64)), (0, new(50, dtype=i64)), (1, new(4)),
                        (1, new(0, dtype=i64)), (2, new(3, dtype=i64)), (2, new(2, 2, dtype=i64)), (2, new(3, 2)),
                        (2, new(3, 1025, dtype=i64)), (3, -1), (3, 65)):
            with pytest.raises(ValueError):
                OPS.policy_log_probs(*(bad if i == at else x for i, x in enumerate(good)))
        for x, rng, p, salt in ((new(3, dtype=i64), new(2, dtype=i64), 0.1, 0), (new(3), new(3, dtype=i64), 0.1, 0),
                                (new(3), new(2), 0.1, 0), (new(3), new(2, dtype=i64), -0.1, 0),
                                (new(3), new(2, dtype=i64), 1.1, 0), (new(3), new(2, dtype=i64), math.nan, 0),
                                (new(3), new(2, dtype=i64), 0.1, -1), (new(3), new(2, dtype=i64), 0.1, 1 << 32)):
            with pytest.raises(ValueError):
                OPS.residual_dropout(x, None, rng, p, salt)


def test_native_argument_checks():
    """What the C entry points refuse, all before any launch: null, unaligned and out-of-range arguments."""
    import ctypes

    from mantisnet import _native

    lib = _native.hip()
    st = (ctypes.c_int64 * 4)(0, 0, 32, 1)
    bad_st = (ctypes.c_int64 * 4)(0, 0, 33, 1)
    P = 4096  # an aligned address that nothing reads

    def forward(**c):
        a = dict(q=P, qs=st, k=P, ks=st, v=P, vs=st, dt=1, bias=P, nb=8, co=P, bu=P, nq=3, nr=3, nl=0, sl=P, n=1, h=1,
                 t=8, hd=32, out=P, os=st, lse=P, stats=P, flag=None, stream=None)
        a.update(c)
        return lib.mantis_relative_attention(*a.values())

    for c in ({"q": None}, {"q": P + 8}, {"out": P + 2}, {"qs": bad_st}, {"os": bad_st}, {"dt": 0}, {"hd": 24},
              {"bias": None}, {"nb": 0}, {"nb": 385}, {"nb": 1, "nl": 1}, {"co": None}, {"co": P + 4}, {"bu": None},
              {"nq": 2}, {"nr": 0}, {"nq": 4097}, {"nq": 65, "nr": 65}, {"nl": -1}, {"nl": 9}, {"h": 0}, {"n": -1},
              {"t": -1}, {"stats": None}, {"stats": P + 4}, {"lse": None}, {"t": 1 << 30}, {"nq": 1 << 33}):
        assert forward(**c) == 1, c
    assert forward(n=0) == 0 and forward(t=0) == 0

    def backward(**c):
        a = dict(q=P, qs=st, k=P, ks=st, v=P, vs=st, go=P, gs=st, stats=P, dt=1, bias=P, nb=8, co=P, bu=P, nq=3, nr=3,
                 nl=0, sl=P, n=1, h=1, t=8, hd=32, ws=P, wsb=1 << 20, dq=P, dqs=st, dk=P, dks=st, dv=P, dvs=st, db=P,
                 flag=None, stream=None)
        a.update(c)
        return lib.mantis_relative_attention_backward(*a.values())

    need = lib.mantis_relative_attention_backward_workspace(1, 1, 8, 8)
    assert need > 0 and lib.mantis_relative_attention_backward_workspace(0, 1, 8, 8) == 0
    for c in ({"go": None}, {"go": P + 4}, {"gs": bad_st}, {"dqs": bad_st}, {"ws": None}, {"wsb": need - 1}, {"db": None},
              {"nb": 385}, {"stats": None}, {"dt": 0}, {"hd": 8}, {"h": 0}):
        assert backward(**c) == 1, c
    assert backward(n=0) == 0

    def policy(**c):
        a = dict(x=P, dt=0, stride=1, off=P, n_pos=2, n=9, mv=P, g=1, top=1, lp=P, en=P, lse=P, tl=P, tm=P, norm=P,
                 ws=None, wsb=0, flag=None, stream=None)
        a.update(c)
        return lib.mantis_policy_log_probs(*a.values())

    for c in ({"x": None}, {"x": P + 2}, {"dt": 3}, {"stride": 0}, {"off": None}, {"n_pos": -1}, {"n": -1}, {"mv": None},
              {"g": -1}, {"g": 1025}, {"top": -1}, {"top": 65}, {"lp": None}, {"tl": None}, {"norm": None},
              {"n_pos": 1, "n": 1 << 20}):  # (a long run needs its workspace)
        assert policy(**c) == 1, c
    assert policy(n_pos=0) == 0 and lib.mantis_policy_log_probs_workspace(1, 1 << 20, 4) > 0

    def dropout(**c):
        a = dict(x=P, dt=0, res=None, rng=P, n=4, p=0.5, salt=0, out=P, odt=0, stream=None)
        a.update(c)
        return lib.mantis_residual_dropout(*a.values())

    for c in ({"x": None}, {"x": P + 2}, {"dt": 3}, {"rng": None}, {"rng": P + 4}, {"n": -1}, {"p": -0.1}, {"p": 1.5},
              {"p": math.nan}, {"salt": -1}, {"salt": 1 << 32}, {"out": None}, {"odt": 3}, {"res": P + 2}):
        assert dropout(**c) == 1, c
    assert dropout(n=0) == 0


def test_reference_gradients_against_differences():
    """The float64 statements the kernels are held to: their gradients along random directions against differences."""
    g = _gen(5)
    case = relative_case([6, 11], 2, 16, torch.float64, 3, n_latents=2)
    q, k, v, bias, coords, buckets, lens, n_latents, grad = case
    val, _amp, _s = relative_reference(q, k, v, bias, coords, buckets, lens, n_latents, grad)
    live = (torch.arange(11)[None] < lens[:, None])[:, None, :, None]
    f = lambda *x: float((relative_reference(*x, coords, buckets, lens, n_latents)[0]["out"] * grad * live).sum())  # noqa: E731
    for at, name in enumerate(("dq", "dk", "dv", "dbias")):
        x = [q, k, v, bias]
        d = torch.randn(x[at].shape, generator=g, dtype=torch.float64)
        up, down = ([y + s * 1e-5 * d if i == at else y for i, y in enumerate(x)] for s in (1, -1))
        assert abs((f(*up) - f(*down)) / 2e-5 - float((val[name] * d).sum())) < 1e-6 * (1 + abs(float((val[name] * d).sum())))
    x = torch.randn(30, generator=g, dtype=torch.float64)
    off, moves = torch.tensor([0, 7, 7, 30]), torch.tensor([[3, 3, -1], [-1, -1, -1], [22, 0, 5]])
    grads = [torch.randn(3, 3, generator=g), torch.randn(3, generator=g), torch.randn(3, generator=g),
             torch.randn(3, 4, generator=g)]
    grads = [y.double() for y in grads]

    def loss(x):
        r = policy_reference(x, off, moves, 4)[0]
        keep = torch.tensor([True, False, True])
        return float((r["log_probs"] * grads[0])[keep].sum() + (r["entropy"] * grads[1])[keep].sum()
                     + (r["lse"] * grads[2])[keep].sum() + (r["top_log_probs"] * grads[3])[keep].sum())

    dx = policy_reference(x, off, moves, 4, grads)[1]
    d = torch.randn(30, generator=g, dtype=torch.float64)
    want = float((dx * d).sum())
    assert abs((loss(x + 1e-6 * d) - loss(x - 1e-6 * d)) / 2e-6 - want) < 1e-6 * (1 + abs(want))


# ----------------------------------------------------------------- GPU: relative attention

BF, HF = torch.bfloat16, torch.float16


@gpu
@pytest.mark.parametrize("lens,heads,d,dtype,kw", [
    ([1], 1, 32, BF, {}),
    ([1, 2, 17], 4, 32, HF, {"n_latents": 0}),
    ([0, 1, 5, 63, 64, 65], 4, 32, BF, {}),
    ([128, 3, 127, 129, 0], 3, 16, HF, {}),
    ([130, 200, 44, 61], 4, 32, BF, {"extra": 5}),
    ([257, 300], 2, 64, HF, {"table": (257, 1), "spread": 150.0}),
    ([333, 64], 2, 64, BF, {"table": (5, 9), "n_latents": 70}),
    ([90, 70], 4, 16, BF, {"n_buckets": 384, "table": (63, 65), "spread": 20.0}),
    ([100, 31], 4, 64, HF, {"n_buckets": 384, "table": (1, 4095), "spread": 900.0}),
    ([80], 2, 32, BF, {"n_buckets": 1, "n_latents": 0, "table": (1, 1)}),
    ([80, 33], 2, 32, HF, {"n_buckets": 2, "n_latents": 40, "table": (1, 3)}),
    ([700, 511, 1021], 2, 32, BF, {"n_buckets": 97}),
    ([40, 20, 9] * 30, 4, 32, BF, {}),
    ([129, 0, 150] * 15, 4, 32, HF, {}),  # 540 tiles of 64 rows: long rows that fill the chip
    ([260, 40, 193] * 12, 3, 16, BF, {"extra": 9, "n_buckets": 384, "table": (63, 65), "spread": 20.0}),
    ([129, 17, 192, 64] * 22, 2, 64, BF, {}),
    ([129, 1, 0, 4, 16, 17, 145], 2, 64, HF, {"n_buckets": 384, "table": (1, 4095), "spread": 900.0}),
])
def test_relative_attention(device, lens, heads, d, dtype, kw):
    case = relative_case(lens, heads, d, dtype, len(lens) + d, device=device, **kw)
    got = check_relative(case)
    ops.raise_on_device_error(device)
    again = _run_relative(case)
    assert all(torch.equal(got[n], again[n]) for n in got)  # the sums run in one order


@gpu
@pytest.mark.parametrize("d", [16, 32, 64])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_relative_attention_reference_point_is_a_score(device, dtype, d):
    # the sum of exp2(c (s - m)) holds the term of m itself, an exact 1, where m is one of the row's
    # scores: its log2 is never below 0; the biases here lie far from the scores
    lens = [*range(1, 68), 80, 81, 112, 113, 128]
    for p, extra in ((1, 0), (len(lens), 0), (len(lens), 13)):
        q, k, v, bias, coords, buckets, sl, n_latents, _grad = relative_case(lens[:p] if p > 1 else [1], 4, d, dtype, 31,
                                                                            device=device, extra=extra)
        case = (2.0 * q, 2.0 * k, v, 4.0 * bias, coords, buckets, sl, n_latents)
        runs = [OPS.fused_attention_relative(*case) for _ in range(4)]
        live = torch.arange(q.shape[2], device=device)[None, None] < sl[:, None, None]
        for out, lse, stats in runs:
            assert bool((stats[..., 1] >= 0)[live.expand(stats.shape[:3])].all())
            assert all(torch.equal(a, b) for a, b in zip((out, lse, stats), runs[0]))
        one = runs[0][2][sl == 1][:, :, 0]
        assert bool((one[..., 1] == 0).all())


@gpu
def test_relative_attention_far_coordinates_and_extents(device):
    # clamped displacements past the table, the coordinates' corners (a difference past int16 saturates)
    case = list(relative_case([50, 50], 2, 32, BF, 3, n_latents=0, table=(9, 5), device=device))
    corners = torch.tensor([[-30000, 30000], [30000, -30000], [0, 0], [30000, 30000], [-30000, -30000]])
    case[4][0, :5] = corners.to(torch.int32).to(device)
    check_relative(case)
    ops.raise_on_device_error(device)


@gpu
@pytest.mark.parametrize("dtype", [BF, HF])
def test_relative_attention_masked_rows(device, dtype):
    # buckets closed by -inf: some rows keep a few keys, some none at all
    q, k, v, bias, coords, buckets, lens, _n, grad = relative_case([70, 20, 129], 4, 32, dtype, 9, n_latents=0,
                                                                   device=device, spread=20.0)
    buckets[:] = 3
    buckets[3, 3] = 5
    bias[:, 3] = -INF
    bias[1, 5] = -INF  # head 1: every key of every row
    coords[0, :10] = 0  # ten stones on one cell see each other; most others only themselves
    case = (q, k, v, bias, coords, buckets, lens, 0, grad)
    got = check_relative(case)
    assert torch.equal(got["lse"][0, 1, :70].cpu(), torch.full((70,), -INF))
    assert not got["out"][0, 1].any() and not got["dq"][0, 1].any() and not got["dv"][0, 1].any()
    assert not got["dbias"][1].any() and not got["dbias"][:, 3].any()


@gpu
def test_relative_attention_lowest_bias(device):
    # a mask of the type's lowest value: beside open keys it weighs 0, alone it is uniform over zero scores
    q, k, v, bias, coords, buckets, lens, _n, grad = relative_case([70, 20], 2, 32, BF, 9, n_latents=0, device=device)
    bias[:, ::2] = torch.finfo(torch.float32).min
    check = (q, k, v, bias, coords, buckets, lens, 0, grad)
    check_relative(check)
    bias[:] = torch.finfo(torch.float32).min
    q = torch.zeros_like(q)  # (fp32 cannot hold a score beside the lowest value)
    got = _run_relative((q, k, v, bias, coords, buckets, lens, 0, grad))
    for i, n in ((0, 70), (1, 20)):
        mean = v[i, :, :n].float().mean(1, keepdim=True).cpu()
        amp = v[i, :, :n].float().abs().mean(1, keepdim=True).cpu()
        _within(got["out"][i, :, :n], mean.expand(-1, n, -1), (2.0**-8 * (3 * amp)).double().expand(-1, n, -1), "out")
        assert torch.equal(got["lse"][i, :, :n].cpu(), torch.full((2, n), torch.finfo(torch.float32).min))
        assert all(bool(got[x].isfinite().all()) for x in ("dq", "dk", "dv", "dbias"))


@gpu
def test_relative_attention_ignores_what_lies_past_the_rows(device):
    case = list(relative_case([30, 1, 64, 0], 2, 32, BF, 21, extra=9, device=device))
    clean = check_relative(case)
    lens = case[6].tolist()
    for x in (case[0], case[1], case[2], case[8]):
        for i, n in enumerate(lens):
            x[i, :, n:] = math.nan
    for i, n in enumerate(lens):
        case[4][i, n:] = 2**31 - 1
    got = _run_relative(case)
    ops.raise_on_device_error(device)
    for name in clean:
        assert torch.equal(clean[name], got[name]), name
    for i, n in enumerate(lens):
        for name in ("out", "dq", "dk", "dv", "lse"):
            assert not got[name][i, :, n:].any()


@gpu
def test_relative_attention_nan_stays(device):
    # a NaN query spoils its own row, a NaN value every row of its position and head that weighs it
    case = list(relative_case([40, 12], 2, 32, HF, 2, device=device))
    case[0][0, 1, 7, 3] = math.nan
    got = _run_relative(case)
    assert got["out"][0, 1, 7].isnan().all() and got["dq"][0, 1, 7].isnan().all()
    assert got["lse"][0, 1, 7].isnan() and not got["out"][0, 0].isnan().any() and not got["out"][1].isnan().any()


@gpu
def test_relative_attention_layouts(device):
    base = relative_case([50, 77, 13], 4, 32, BF, 4, device=device)
    q, k, v, bias, coords, buckets, lens, n_latents, grad = base
    want = _run_relative(tuple(x.contiguous() if isinstance(x, torch.Tensor) else x for x in base))
    p, a, t, d = q.shape
    packed = torch.stack([x.transpose(1, 2) for x in (q, k, v)], 2).contiguous()  # (P, T, 3, A, D)
    forms = [
        [packed[:, :, j].transpose(1, 2) for j in range(3)],
        # rows that start off a 16-byte boundary, and a dimension that is not innermost
        [torch.cat([x.reshape(-1).new_zeros(3), x.reshape(-1)])[3:].view(x.shape) for x in (q, k, v)],
        [x.transpose(2, 3).contiguous().transpose(2, 3) for x in (q, k, v)],
    ]
    for qkv in forms:
        leaves = [x.requires_grad_(True) for x in (*[y.detach() for y in qkv], bias.detach())]
        out, lse, _ = OPS.fused_attention_relative(*leaves, coords, buckets, lens, n_latents)
        g = torch.autograd.grad(out, leaves, grad.transpose(2, 3).contiguous().transpose(2, 3))
        for name, x in zip(("out", "lse", "dq", "dk", "dv", "dbias"), (out, lse, *g)):
            assert torch.equal(x, want[name]), name
    # one head's rows for every head, and a gradient that is one number everywhere
    one = q[:, :1].expand(p, a, t, d)
    leaf = q[:, :1].detach().requires_grad_(True)
    out, _, _ = OPS.fused_attention_relative(leaf.expand(p, a, t, d), k, v, bias, coords, buckets, lens, n_latents)
    (d1,) = torch.autograd.grad(out.sum(), leaf)
    val, amp, score = relative_reference(one, k, v, bias, coords, buckets, lens, n_latents, torch.ones_like(q))
    tol = _relative_tolerances(val, amp, score, BF, t, d, 6)["dq"].sum(1, keepdim=True)
    _within(d1, val["dq"].sum(1, keepdim=True), tol + 5 * HALF_STEP[BF] * val["dq"].abs().sum(1, keepdim=True), "shared head")
    # dimensions of one entry report any stride
    single = [x[:1, :1, :1].contiguous().as_strided((1, 1, 1, d), (7, 3, 5, 1)) for x in (q, k, v)]
    out, lse, _ = OPS.fused_attention_relative(*single, bias[:1], coords[:1, :1], buckets,
                                               torch.ones(1, dtype=torch.int32, device=device), 1)
    assert torch.equal(out, single[2])


@gpu
def test_relative_attention_types_of_bias_and_empty_batches(device):
    q, k, v, bias, coords, buckets, lens, n_latents, grad = relative_case([20, 9], 2, 16, HF, 6, device=device)
    half = bias.bfloat16().requires_grad_(True)
    out, _, _ = OPS.fused_attention_relative(q, k, v, half, coords, buckets, lens, n_latents)
    (db,) = torch.autograd.grad(out, half, grad)
    want = _run_relative((q, k, v, half.detach().float(), coords, buckets, lens, n_latents, grad))
    assert db.dtype == torch.bfloat16 and torch.equal(db, want["dbias"].bfloat16())
    for shape in ((0, 2, 9, 16), (3, 2, 0, 16)):
        leaves = [torch.zeros(shape, dtype=HF, device=device, requires_grad=True) for _ in range(3)]
        b = bias.detach().requires_grad_(True)
        out, lse, _ = OPS.fused_attention_relative(
            *leaves, b, torch.zeros(shape[0], shape[2], 2, dtype=torch.int32, device=device), buckets,
            torch.zeros(shape[0], dtype=torch.int32, device=device), 0)
        g = torch.autograd.grad(out.sum(), [*leaves, b])
        assert out.shape == shape and lse.shape == shape[:3] and not g[3].any()


@gpu
def test_relative_attention_flags(device):
    case = list(relative_case([20, 9], 2, 16, HF, 6, device=device))
    case[5][0, 0] = 12  # one past the last bucket: no bias, no gradient
    case[5][6, 1] = -3
    got = _run_relative(case)
    with pytest.raises(ValueError, match="out of range"):
        ops.raise_on_device_error(device)
    q, k, v, bias, coords, buckets, lens, n_latents, grad = case
    val, amp, score = relative_reference(q, k, v, bias, coords, buckets, lens, n_latents, grad)
    tol = _relative_tolerances(val, amp, score, HF, 20, 16, 2)
    for name in got:
        _within(got[name], val[name], tol[name], name)
    case = list(relative_case([20, 9], 2, 16, HF, 6, device=device))
    case[4][0, 10, 1] = 40000
    _run_relative(case)
    with pytest.raises(ValueError, match="out of range"):
        ops.raise_on_device_error(device)


# ----------------------------------------------------------------- GPU: policy


def policy_case(lens, dtype, seed, device, *, moves=2, top=4, scale=2.0, step=0.0, lead=0, tail=0):
    g = _gen(seed)
    offsets = torch.tensor([lead] + [lead + sum(lens[:i + 1]) for i in range(len(lens))])
    x = torch.randn(int(offsets[-1]) + tail, generator=g) * scale
    if step:
        x = (x / step).round() * step  # ties
    n = torch.tensor(lens)[:, None]
    mv = (torch.rand(len(lens), moves, generator=g) * n).long().clamp(max=(n - 1).clamp(min=0))
    mv = torch.where(n > 0, mv, -1)
    p = len(lens)
    grads = [torch.randn(s, generator=g).to(device) for s in ((p, moves), (p,), (p,), (p, top))]
    return x.to(dtype).to(device), offsets.to(device), mv.to(device), top, grads


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, BF, HF])
@pytest.mark.parametrize("lens,kw", [
    ([1], {"top": 1, "moves": 1}),
    ([5, 0, 1, 2], {"top": 8}),
    ([63, 64, 65, 255, 256, 257], {"top": 64, "moves": 7}),
    ([300, 1200, 7, 1023, 1024, 1025], {"step": 0.5, "top": 16}),
    ([5000, 1], {"top": 32, "lead": 3, "tail": 5}),
    ([70001, 33], {"step": 0.25, "top": 5}),
    ([200003], {"top": 64, "moves": 33, "tail": 1}),
    ([9000, 10007, 8191], {"top": 0, "moves": 0}),
    ([30] * 700, {"top": 3, "moves": 1}),
])
def test_policy_log_probs(device, dtype, lens, kw):
    check_policy(*policy_case(lens, dtype, len(lens), device, **kw))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, BF])
def test_policy_masked_and_broken_runs(device, dtype):
    x, off, mv, top, grads = policy_case([40, 40, 40, 40, 40, 40, 0, 12000, 12000], dtype, 8, device, top=8, moves=3)
    x[0:30] = -INF  # ten possible moves
    x[40:80] = -INF  # none
    x[85] = math.nan
    x[125] = INF
    x[160:200] = torch.finfo(dtype).min  # uniform over the lowest value
    x[200:230] = torch.finfo(dtype).min
    x[240:12200] = -INF  # a sliced run with 40 possible moves
    x[13000] = math.nan
    mv[0] = torch.tensor([3, 35, 3])  # a closed move, an open one, the closed one again
    mv[1] = torch.tensor([3, -1, 5])
    check_policy(x, off, mv, top, grads)


@gpu
def test_policy_equal_logits_take_the_lowest_indices(device):
    x = torch.zeros(3000 + 20000, device=device)
    out = OPS.policy_log_probs(x, torch.tensor([0, 3000, 23000], device=device),
                               torch.zeros(2, 0, dtype=torch.long, device=device), 64)
    assert torch.equal(out[4].cpu(), torch.arange(64).expand(2, 64))
    rising = torch.arange(23000.0, device=device) / 4096  # every entry beats all before it
    out = OPS.policy_log_probs(rising, torch.tensor([0, 3000, 23000], device=device),
                               torch.zeros(2, 0, dtype=torch.long, device=device), 10)
    assert torch.equal(out[4].cpu(), torch.stack([2999 - torch.arange(10), 19999 - torch.arange(10)]))


@gpu
def test_policy_strides_offsets_and_missing_gradients(device):
    x, off, mv, top, grads = policy_case([50, 333, 8000, 70000], torch.float32, 12, device, top=6)
    rows = torch.randn(x.numel(), 4, device=device)
    rows[:, 1] = x
    check_policy(rows[:, 1], off, mv, top, grads)
    for keep in range(4):
        check_policy(x, off, mv, top, [g if i == keep else None for i, g in enumerate(grads)])
    # large common offsets cost the log probabilities nothing
    check_policy(x.round() + 4096.0, off, mv, top, grads)
    half = torch.cat([x.new_zeros(1), x]).half()[1:]  # two bytes past an aligned address
    check_policy(half, off, mv, top, grads)


@gpu
def test_policy_bad_moves_and_offsets(device):
    x, off, mv, top, grads = policy_case([50, 33], torch.float32, 12, device, top=6)
    mv[0, 0], mv[1, 1] = 50, -2
    check_policy(x, off, mv, top, grads, need_error=True)
    for bad in ([0, 60, 50], [-1, 50, 83], [0, 50, 84]):
        OPS.policy_log_probs(x, torch.tensor(bad, device=device), torch.full_like(mv, -1), top)
        with pytest.raises(ValueError, match="not ascending"):
            ops.raise_on_device_error(device)
    none = OPS.policy_log_probs(x[:0], torch.zeros(3, dtype=torch.long, device=device), torch.full_like(mv, -1), 2)
    assert torch.equal(none[2].cpu(), torch.full((2,), -INF)) and not none[1].any()
    assert torch.equal(none[4].cpu(), torch.full((2, 2), -1))
    leaf = x.clone().requires_grad_(True)
    out = OPS.policy_log_probs(leaf, torch.zeros(1, dtype=torch.long, device=device), mv[:0], 2)
    (dx,) = torch.autograd.grad(out[1].sum(), leaf)
    assert out[0].shape == (0, 2) and not dx.any()


# ----------------------------------------------------------------- GPU: dropout


def _dropout_reference(x, residual, rng, p, salt):
    words = philox_words(x.numel(), *rng, salt)
    keep = torch.from_numpy(words >= np.uint64(min(round(p * 2**32), 2**32))).view(x.shape)
    scaled = torch.where(keep, x.double() / (1 - p) if p < 1 else 0.0, 0.0)
    return keep, scaled if residual is None else residual.double() + scaled


@gpu
@pytest.mark.parametrize("x_dtype,r_dtype", [(a, b) for a in (torch.float32, BF, HF) for b in (None, torch.float32, BF, HF)])
@pytest.mark.parametrize("shape,p", [((1,), 0.5), ((3, 7), 0.1), ((5, 128), 0.25), ((1021, 3), 0.9), ((2, 3, 5), 0.0),
                                     ((4, 4), 1.0)])
def test_residual_dropout(device, x_dtype, r_dtype, shape, p):
    g = _gen(3)
    x = torch.randn(shape, generator=g).to(x_dtype)
    res = None if r_dtype is None else torch.randn(shape, generator=g).to(r_dtype)
    rng, salt = (0x0123456789ABCDEF, (1 << 33) + 7), 0xFFFFFFFF
    leaves = [t.to(device).requires_grad_(True) for t in (x, res) if t is not None]
    state = torch.tensor(rng, device=device)
    out = OPS.residual_dropout(leaves[0], leaves[1] if res is not None else None, state, p, salt)
    grad = torch.randn(shape, generator=g).to(out.dtype)
    grads = torch.autograd.grad(out, leaves, grad.to(device))
    keep, want = _dropout_reference(x, res, rng, p, salt)
    tiny = lambda dt: 2.0**-25 if dt == torch.float16 else 0.0  # noqa: E731
    # the scale rounds to fp32, the sum to fp32 and to its type
    tol = (2.0**-24 + HALF_STEP[out.dtype]) * want.abs() + 2.0**-23 * (want - (0 if res is None else res.double())).abs()
    _within(out, want, tol + tiny(out.dtype), "out")
    dx = torch.where(keep, grad.double() / (1 - p) if p < 1 else 0.0, 0.0)
    _within(grads[0], dx, (2.0**-23 + HALF_STEP[x_dtype]) * dx.abs() + tiny(x_dtype), "dx")
    assert grads[0].dtype == x_dtype and (res is None or torch.equal(grads[1].cpu(), grad))


@gpu
def test_residual_dropout_layouts_and_specials(device):
    state = torch.tensor([9, 2], device=device)
    x = torch.randn(64, 130, device=device)
    want = OPS.residual_dropout(x, None, state, 0.5, 1)
    assert torch.equal(OPS.residual_dropout(x.t().contiguous().t(), None, state, 0.5, 1), want)  # row-major order
    flat = torch.cat([x.new_zeros(1), x.reshape(-1)])[1:]  # four bytes past an aligned address
    assert torch.equal(OPS.residual_dropout(flat, flat, state, 0.5, 1), OPS.residual_dropout(
        flat.clone(), flat.clone(), state, 0.5, 1))
    keep = want != 0
    assert 0.45 < float(keep.float().mean()) < 0.55
    bad = torch.where(keep, x, math.nan)  # what is dropped does not spread
    assert torch.equal(OPS.residual_dropout(bad, None, state, 0.5, 1), want)
    assert OPS.residual_dropout(torch.where(keep, math.nan, x), None, state, 0.5, 1).isnan().equal(keep)
    for other, salt in ((state + torch.tensor([0, 1], device=device), 1), (state, 2),
                        (state + torch.tensor([1, 0], device=device), 1)):
        agree = (OPS.residual_dropout(x, None, other, 0.5, salt) != 0).eq(keep).float().mean()
        assert 0.45 < float(agree) < 0.55  # another step, salt or seed: another mask
    assert OPS.residual_dropout(x[:0], None, state, 0.5, 1).shape == (0, 130)
    leaf = x.clone().requires_grad_(True)
    out = OPS.residual_dropout(leaf, None, state, 0.5, 1)
    state += 1
    with pytest.raises(RuntimeError, match="inplace"):
        out.sum().backward()
    with pytest.raises(ValueError):
        OPS.residual_dropout(x, x[:1], state, 0.5, 1)


# ----------------------------------------------------------------- GPU: together


def _block(p, x, extra):
    """One training step of a small block: attention with the relative bias onto
    its residual under dropout, a policy row per stone, the loss of the moves played."""
    coords, buckets, lens, rng, offsets, moves = extra
    n, t, h = x.shape
    qkv = (x.to(BF) @ p["qkv"].to(BF)).view(n, t, 3, 4, 32)
    q, k, v = (qkv[:, :, j].transpose(1, 2) for j in range(3))
    out, _, _ = OPS.fused_attention_relative(q, k, v, p["bias"], coords, buckets, lens, 4)
    y = OPS.residual_dropout(out.transpose(1, 2).reshape(n, t, h) @ p["wo"].to(BF), x, rng, 0.1, 3)
    logits = (y @ p["head"]).view(-1)
    log_probs, entropy, *_ = OPS.policy_log_probs(logits, offsets, moves, 0)
    return -log_probs.mean() - 0.01 * entropy.mean()


def _block_case(device):
    g = _gen(1)
    new = lambda *s, scale=1.0: (torch.randn(s, generator=g) * scale).to(device)  # noqa: E731
    lens = torch.tensor([44, 61, 9], dtype=torch.int32, device=device)
    t = 64
    buckets, count = tables.relative_buckets(5)
    params = {"qkv": new(128, 384, scale=0.09), "wo": new(128, 128, scale=0.09), "head": new(128, 1, scale=0.1),
              "bias": new(4, count)}
    x = new(3, t, 128)
    extra = ((torch.randn(3, t, 2, generator=g) * 4).round().to(torch.int32).to(device), buckets.to(device), lens,
             torch.tensor([77, 0], device=device), torch.tensor([0, t, 2 * t, 3 * t], device=device),
             torch.tensor([[4, 9], [11, -1], [5, 5]], device=device))
    return params, x, extra


def _block_reference(params, x, extra):
    """The same step in float64 (16-bit operands rounded where the step rounds them are not)."""
    coords, buckets, lens, rng, offsets, moves = (e.cpu() for e in extra)
    p = {k: w.detach().cpu().double().requires_grad_(True) for k, w in params.items()}
    x = x.detach().cpu().double()
    n, t, h = x.shape
    q, k, v = ((x @ p["qkv"]).view(n, t, 3, 4, 32)[:, :, j].transpose(1, 2) for j in range(3))
    att = []
    for i in range(n):
        m = int(lens[i])
        pair = _pairs(coords[i], buckets, m, 4, p["bias"].shape[1])
        s = q[i, :, :m] @ k[i, :, :m].transpose(1, 2) / math.sqrt(32) + p["bias"][:, pair]
        att.append(torch.cat([s.softmax(2) @ v[i, :, :m], torch.zeros(4, t - m, 32)], 1))
    keep = torch.from_numpy(philox_words(x.numel(), *rng.tolist(), 3) >= np.uint64(round(0.1 * 2**32))).view(x.shape)
    y = x + torch.where(keep, (torch.stack(att).transpose(1, 2).reshape(n, t, h) @ p["wo"]) / 0.9, 0.0)
    logp = (y @ p["head"]).view(n, t).log_softmax(1)
    played = torch.where(moves >= 0, logp.gather(1, moves.clamp(min=0)), 0.0)
    loss = -played.mean() + 0.01 * (logp.exp() * logp).sum(1).mean()
    return loss, torch.autograd.grad(loss, list(p.values()))


@gpu
def test_a_training_step_of_all_three(device):
    params, x, extra = _block_case(device)
    leaves = {k: w.clone().requires_grad_(True) for k, w in params.items()}
    loss = _block(leaves, x, extra)
    grads = torch.autograd.grad(loss, list(leaves.values()))
    ops.raise_on_device_error(device)
    want, exact = _block_reference(params, x, extra)
    # bf16 operands at five places between the input and the loss, each half a
    # step relative to the values there: in the 2-norm 8 half steps of bf16
    assert abs(float(loss.detach()) - float(want.detach())) < 8 * 2.0**-8 * (1 + abs(float(want.detach())))
    for name, g, e in zip(params, grads, exact):
        assert float((g.cpu().double() - e).norm()) < 8 * 2.0**-8 * float(e.norm()), name


@gpu
def test_a_captured_step_replays_with_another_mask(device):
    params, x, extra = _block_case(device)
    leaves = {k: w.clone().requires_grad_(True) for k, w in params.items()}
    rng = extra[3]

    def step():
        loss = _block(leaves, x, extra)
        return [loss.detach(), *torch.autograd.grad(loss, list(leaves.values()))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # (also: another stream than the inputs' own)
        eager = step()
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    first = None
    for replay in range(4):
        rng.copy_(torch.tensor([77, replay // 2]))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        for got, exp in zip(held, want):
            assert torch.equal(got, exp), replay
        if replay == 0:
            first = [h.clone() for h in held]
            assert all(torch.equal(a, b) for a, b in zip(first, eager))
        elif replay == 2:
            assert not torch.equal(first[0], held[0])  # another step, another mask
    ops.raise_on_device_error(device)


@gpu
def test_calls_on_two_streams_and_graphs_side_by_side(device):
    # long rows of one position (tiles of 16 rows), a sliced run: the calls with workspaces
    cases = [relative_case([300, 257], 2, 32, BF, s, device=device) for s in (1, 2)]
    logits = [torch.randn(2 * 30000, generator=_gen(s)).to(device) for s in (3, 4)]
    offsets = torch.tensor([0, 30000, 60000], device=device)
    moves = torch.tensor([[7, 29999], [0, -1]], device=device)

    def step(i):
        leaf = logits[i].detach().requires_grad_(True)
        log_probs, entropy, lse, top, _moves, _norm = OPS.policy_log_probs(leaf, offsets, moves, 5)
        (grad,) = torch.autograd.grad(log_probs.sum() + entropy.sum() + top.sum(), leaf)
        return [*_run_relative(cases[i]).values(), log_probs.detach(), lse.detach(), grad]

    want = [step(0), step(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got = []
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got.append(step(i))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))
    graphs, held = [], []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            held.append(step(i))
    for _ in range(3):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for h, w in zip(held, want) for a, b in zip(h, w))
    ops.raise_on_device_error(device)


@gpu
def test_relative_attention_positions_further_apart_than_32_bits(device):
    q, k, v, bias, coords, buckets, lens, n_latents, grad = relative_case([20, 17], 2, 16, BF, 12, device=device)
    apart = 2**31 + 8  # elements: more than 2^32 bytes
    far = torch.empty(apart + q[0].numel(), dtype=BF, device=device).as_strided(q.shape, (apart, *q.stride()[1:]))
    far.copy_(q)
    got = _run_relative((q, k, v, bias, coords, buckets, lens, n_latents, grad))
    for at in range(3):
        ops3 = [q, k, v]
        ops3[at] = far.copy_(ops3[at])
        out, lse, stats = OPS.fused_attention_relative(*ops3, bias, coords, buckets, lens, n_latents)
        dq, dk, dv, dbias = OPS.fused_attention_relative_backward(*ops3, bias, coords, buckets, lens, n_latents, stats,
                                                                  grad)
        for name, x in zip(("out", "lse", "dq", "dk", "dv", "dbias"), (out, lse, dq, dk, dv, dbias)):
            assert torch.equal(x, got[name]), (at, name)


@gpu
def test_backwards_are_not_differentiable(device):
    q, k, v, bias, coords, buckets, lens, n_latents, grad = relative_case([9], 1, 16, BF, 13, device=device)
    leaf = q.clone().requires_grad_(True)
    out, _, _ = OPS.fused_attention_relative(leaf, k, v, bias, coords, buckets, lens, n_latents)
    x = torch.randn(6, device=device, requires_grad=True)
    log_probs = OPS.policy_log_probs(x, torch.tensor([0, 6], device=device), torch.tensor([[2]], device=device), 0)[0]
    y = OPS.residual_dropout(x, None, torch.tensor([1, 2], device=device), 0.5, 0)
    for result, wrt in ((out, leaf), (log_probs, x), (y, x)):
        weight = torch.ones_like(result, requires_grad=True)
        (first,) = torch.autograd.grad(result, wrt, weight, create_graph=True)
        with pytest.raises(RuntimeError, match="not implemented"):
            first.sum().backward()
