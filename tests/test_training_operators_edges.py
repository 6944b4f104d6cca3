"""Edges of the training operators: layouts and traces of their results, infinite
and cancelling gradients, broken index tables, the library's absence.

The formulas in float64 and the tolerances are those of
``test_training_operators.py`` unless a test states its own.
"""

from __future__ import annotations

import math
import os
import shutil
import subprocess
import sys
import threading
from pathlib import Path

import pytest
import torch

import mantisnet
from mantisnet import ops, tables
from tests import test_training_operators as base

OPS, INF, BF, HF = base.OPS, base.INF, base.BF, base.HF
gpu = base.gpu


# ----------------------------------------------------------------- layouts of results


def _layouts(p, a, t, d, new):
    """Operands (P, A, T, D) as programs hold them, and the order (outermost first) of their results' memory."""
    rows, heads = (0, 2, 1, 3), (0, 1, 2, 3)
    return {
        "contiguous": (new(p, a, t, d), heads),
        "projection": (new(p, t, a, d).transpose(1, 2), rows),
        "packed": (new(p, t, 3, a, d)[:, :, 1].transpose(1, 2), rows),
        "packed first": (new(3, p, t, a, d)[2].transpose(1, 2), rows),
        "sliced": (new(p, a, t, 2 * d)[..., :d], heads),
        "every other row": (new(p, 2 * t, a, d)[:, ::2].transpose(1, 2), rows),
        "heads outermost": (new(a, t + 3, p, d)[:, 3:].permute(2, 0, 1, 3), (1, 2, 0, 3)),
        "shared head": (new(p, 1, t, d).expand(p, a, t, d), heads),
        "shared position": (new(1, t, a, d).transpose(1, 2).expand(p, a, t, d), heads if p > 1 else rows),
        "not innermost": (new(p, a, d, t).transpose(2, 3), heads),
        "far rows": (new(p, t, 8200).as_strided((p, a, t, d), (t * 8200, d, 8200, 1)), rows),
    }


def _dense(shape, order):
    strides, step = [0] * 4, 1
    for i in reversed(order):
        strides[i] = step
        step *= shape[i]
    return tuple(strides)


def _relative_on(q, new, i32):
    p, a, t, _ = q.shape
    return (q, q, q, new(a, 12), i32(p, t, 2), i32(5, 7), i32(p), min(4, t))


def test_fake_results_lie_in_their_operands_order():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        half = lambda *s: torch.empty(s, dtype=BF, device="cuda")  # noqa: E731
        new = lambda *s: torch.empty(s, device="cuda")  # noqa: E731
        i32 = lambda *s: torch.empty(s, dtype=torch.int32, device="cuda")  # noqa: E731
        for shape in ((2, 4, 64, 32), (3, 2, 1, 16), (1, 4, 9, 64), (5, 1, 7, 16)):
            for name, (q, order) in _layouts(*shape, half).items():
                out, lse, stats = OPS.fused_attention_relative(*_relative_on(q, new, i32))
                want = _dense(shape, order)
                for x in (out, *OPS.fused_attention_relative_backward(*_relative_on(q, new, i32), stats, q)[:3]):
                    assert x.shape == shape
                    assert all(n == 1 or s == w for n, s, w in zip(shape, x.stride(), want)), (name, shape, x.stride())
                assert lse.is_contiguous() and stats.is_contiguous()
        # 256 heads of 64 in a row: past the kernels' pitch
        wide, _ = _layouts(2, 256, 5, 64, half)["projection"]
        assert OPS.fused_attention_relative(*_relative_on(wide, new, i32))[0].is_contiguous()


def _fakes_of(mode, xs):
    return [mode.from_tensor(x) if isinstance(x, torch.Tensor) else x for x in xs]


@gpu
def test_results_lie_where_their_fakes_say(device):
    from torch._subclasses.fake_tensor import FakeTensorMode

    def agree(op, *args):
        res = op(*args)
        mode = FakeTensorMode()
        with mode:
            fake = op(*_fakes_of(mode, args))
        for r, f in zip(res if isinstance(res, tuple) else [res], fake if isinstance(fake, tuple) else [fake]):
            assert (r.shape, r.stride(), r.dtype, r.device) == (f.shape, f.stride(), f.dtype, f.device), op
        return res

    for shape in ((2, 4, 64, 32), (3, 2, 1, 16), (1, 2, 200, 64)):
        p, a, t, _ = shape
        _q, _k, _v, bias, coords, buckets, _l, _n, _g = base.relative_case([t] * p, a, shape[3], BF, 3, device=device)
        lens = torch.randint(0, t + 1, (p,), dtype=torch.int32, device=device)
        half = lambda *s: torch.randn(s, device=device).to(BF)  # noqa: E731
        for q, _order in _layouts(*shape, half).values():
            args = (q, q, q, bias, coords, buckets, lens, min(4, t))
            out, _lse, stats = agree(OPS.fused_attention_relative, *args)
            grads = agree(OPS.fused_attention_relative_backward, *args, stats, out)
            plain = tuple(x.contiguous() if isinstance(x, torch.Tensor) else x for x in args)
            assert torch.equal(out, OPS.fused_attention_relative(*plain)[0])
            for x, y in zip(grads, OPS.fused_attention_relative_backward(*plain, stats, out.contiguous())):
                assert torch.equal(x, y)
    x, off, mv, top, grads = base.policy_case([50, 333], BF, 12, device, top=6)
    for logits in (x, torch.stack([x, x], 1)[:, 1], x[:1].expand(x.numel())):
        res = agree(OPS.policy_log_probs, logits, off, mv, top)
        agree(OPS.policy_log_probs_backward, logits, off, mv, res[4], res[1], res[5], *grads)
    rng = torch.tensor([3, 4], device=device)
    for y in (torch.randn(6, 10, device=device), torch.randn(10, 6, device=device).t()):
        out = agree(OPS.residual_dropout, y, y.half(), rng, 0.1, 2)
        agree(OPS.residual_dropout_backward, out, rng, 0.1, 2, BF)


@gpu
def test_a_traced_step_over_packed_rows(device):
    from torch.fx.experimental.proxy_tensor import make_fx

    params, x, extra = base._block_case(device)
    leaves = [w.clone().requires_grad_(True) for w in params.values()]

    def step(*leaves):
        loss = base._block(dict(zip(params, leaves)), x, extra)
        return loss, *torch.autograd.grad(loss, leaves)

    want = step(*leaves)
    traced = make_fx(step, tracing_mode="fake", _allow_non_fake_inputs=True)(*leaves)
    got = traced(*[w.detach() for w in leaves])
    for name, g, w in zip(("loss", *params), got, want):
        assert torch.equal(g.detach(), w.detach()), name


def _block_args(device, positions=6, t=61):
    params, x, (coords, buckets, lens, rng, _offsets, _moves) = base._block_case("cpu")
    x = torch.randn(positions, t, 128, generator=base._gen(t))
    coords = (torch.randn(positions, t, 2, generator=base._gen(t + 1)) * 4).round().to(torch.int32)
    lens = torch.randint(4, t + 1, (positions,), generator=base._gen(t + 2)).to(torch.int32)
    moves = torch.randint(0, t, (positions, 2), generator=base._gen(t + 3))
    extra = (coords, buckets, lens, rng, torch.arange(positions + 1) * t, moves)
    leaves = [w.to(device).requires_grad_(True) for w in params.values()]
    return list(params), leaves, x.to(device), [e.to(device) for e in extra]


def test_a_step_traces_with_open_sizes():
    from torch.fx.experimental.proxy_tensor import make_fx

    names, leaves, x, extra = _block_args("meta")

    def step(x, extra, *leaves):
        loss = base._block(dict(zip(names, leaves)), x, extra)
        return loss, *torch.autograd.grad(loss, leaves)

    graph = make_fx(step, tracing_mode="symbolic")(x, extra, *leaves)
    shapes = {}
    for node in graph.graph.nodes:
        if "mantisnet" in str(node.target):
            val = node.meta["val"]
            shapes[node.target._opname] = (val[0] if isinstance(val, (tuple, list)) else val).shape
    assert set(shapes) == set(base.NAMES)
    for name, shape in shapes.items():  # the batch and the rows stay open
        assert not isinstance(shape[0], int), name
    assert not isinstance(shapes["fused_attention_relative"][2], int)


@gpu
def test_a_compiled_step_takes_other_sizes(device):
    names, _, _, _ = _block_args("cpu")

    def loss_of(leaves, x, extra):
        return base._block(dict(zip(names, leaves)), x, extra)

    torch._dynamo.reset()
    graphs = []

    def backend(gm, example):
        from torch._dynamo.backends.common import aot_autograd

        graphs.append(gm)
        return aot_autograd(fw_compiler=lambda g, _: g)(gm, example)

    compiled = torch.compile(loss_of, backend=backend, dynamic=True, fullgraph=True)
    for positions, t in ((6, 61), (9, 37), (5, 150)):  # (no other size is one of these: equal sizes share a symbol)
        _, leaves, x, extra = _block_args(device, positions, t)
        got = torch.autograd.grad(compiled(leaves, x, extra), leaves)
        want = torch.autograd.grad(loss_of(leaves, x, extra), leaves)
        for name, g, w in zip(names, got, want):
            assert torch.equal(g, w), (name, positions, t)
    assert len(graphs) == 1
    torch._dynamo.reset()


# ----------------------------------------------------------------- infinite operands


@gpu
@pytest.mark.parametrize("lens", [[1, 2, 3, 40, 128], [1, 2, 150], [200, 3, 1, 129] * 4])
@pytest.mark.parametrize("d", [16, 32, 64])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_relative_attention_infinite_gradients_and_values(device, dtype, d, lens):
    """An infinite entry gives infinities and NaNs where the formula does: an infinite incoming
    gradient infinite dv, an infinite value infinite outputs and, where its row's signs agree, dk."""
    q, k, v, bias, coords, buckets, sl, n_latents, grad = base.relative_case(lens, 4, d, dtype, 17, device=device)
    for i, n in enumerate(lens):
        grad[i, 1, n - 1, 3] = INF
        grad[i, 2, n // 2, 5] = -INF
        v[i, 3, n - 1, 2] = INF
    case = (q, k, v, bias, coords, buckets, sl, n_latents, grad)
    got = base._run_relative(case)
    val, amp, score = base.relative_reference(*case)
    tol = base._relative_tolerances(val, amp, score, dtype, q.shape[2], d, len(lens) * 4)
    for name in got:
        x, exp = got[name].detach().cpu().double(), val[name]
        assert torch.equal(x.isnan(), exp.isnan()), name
        assert torch.equal(x[exp.isinf()], exp[exp.isinf()]), name
        base._within(got[name], exp, tol[name].nan_to_num(0.0), name)
    assert (val["dv"] == INF).any() and (val["dv"] == -INF).any() and val["dk"].isinf().any()
    assert val["out"].isinf().any() and not val["dv"][:, 0].isinf().any()


# ----------------------------------------------------------------- gradients whose terms cancel


def _elementwise(q, k, v, bias, pair, grad, dtype):
    """(dq, dk, p, dp - delta) of one position and head, the formula in ``dtype``."""
    q, k, v, bias, grad = (x.to(dtype) for x in (q, k, v, bias, grad))
    s = q @ k.T / math.sqrt(q.shape[1]) + bias[pair]
    p = torch.exp(s - s.amax(1, keepdim=True))
    p = p / p.sum(1, keepdim=True)
    dp = grad @ v.T
    off = dp - (p * dp).sum(1, keepdim=True)
    ds = p * off
    return ds @ k / math.sqrt(q.shape[1]), ds.T @ q / math.sqrt(q.shape[1]), p, off


@gpu
@pytest.mark.parametrize("lens,extra", [([100, 128, 65], 0), ([100, 128, 65], 40), ([300, 129, 512], 0),
                                        ([300, 140, 512] * 6, 0)])
@pytest.mark.parametrize("kind", ["peaked", "sharp", "offset", "twins"])
@pytest.mark.parametrize("dtype,d", [(BF, 16), (BF, 32), (BF, 64), (HF, 32), (HF, 64)])
def test_relative_attention_gradients_that_cancel(device, dtype, d, kind, lens, extra):
    """dq and dk where dp - delta is far smaller than dp: rows that one key holds (all but 1e-3 or
    1e-5 of the weight), keys and values with a mean of many deviations, equal keys.

    In the 2-norm over a head, the error is at most the output's half step, three times the
    error of the fp32 formula on the same inputs (the same roundings in another order), and the
    cut of the parts: 2^-16 of the terms p |dp - delta| |k| and, for what r moves past, of their
    row sums times sum p |k|."""
    q, k, v, bias, coords, buckets, sl, _n, grad = base.relative_case(lens, 2, d, dtype, 23, n_latents=0, extra=extra,
                                                                     device="cpu")
    g = base._gen(3)
    t = q.shape[2]
    if kind in ("peaked", "sharp"):  # a row's own key stands out of the others by its score
        gap = 10.0 if kind == "peaked" else 16.0
        q = (torch.randn(q.shape, generator=g) * 0.5).to(dtype)
        u = torch.nn.functional.normalize(torch.randn(len(lens), 2, t, d, generator=g), dim=3)
        q, k = (u * gap).to(dtype), (u * math.sqrt(d)).to(dtype)
        bias.zero_()
    elif kind == "offset":
        mean = 40.0 if dtype == HF else 160.0
        k = (k.float() + mean * torch.randn(2, 1, d, generator=g).sign()).to(dtype)
        v = (v.float() + mean * torch.randn(2, 1, d, generator=g).sign()).to(dtype)
    else:  # two equal keys hold a row between them
        u = torch.nn.functional.normalize(torch.randn(len(lens), 2, t, d, generator=g), dim=3)
        u[:, :, 1::2] = u[:, :, 0:t - t % 2:2]
        v = v.clone()
        v[:, :, 1::2] = v[:, :, 0:t - t % 2:2]
        q, k = (u * 14.0).to(dtype), (u * math.sqrt(d)).to(dtype)
        bias.zero_()
    case = [x.to(device) for x in (q, k, v, bias, coords, buckets, sl)] + [0, grad.to(device)]
    got = base._run_relative(tuple(case))
    u16 = base.HALF_STEP[dtype]
    least = 2.0**-25 if dtype == HF else 0.0
    for h in range(2):
        sums = {n: [0.0] * 4 for n in ("dq", "dk")}
        for i, n in enumerate(lens):
            pair = base._pairs(coords[i], buckets, n, 0, bias.shape[1])
            one = [x[i, h, :n] for x in (q, k, v)] + [bias[h], pair, grad[i, h, :n]]
            dq, dk, p, off = _elementwise(*one, torch.float64)
            dq32, dk32, _, _ = _elementwise(*one, torch.float32)
            ka, qa = k[i, h, :n].double().abs(), q[i, h, :n].double().abs()
            terms = p * off.abs()
            cut = {"dq": terms @ ka + terms.sum(1, keepdim=True) * (p @ ka), "dk": terms.T @ qa}
            for name, exp, low in (("dq", dq, dq32), ("dk", dk, dk32)):
                x = got[name][i, h, :n].cpu().double()
                for j, y in enumerate((x - exp, exp, low.double() - exp, cut[name] / math.sqrt(d))):
                    sums[name][j] += float(y.square().sum())
        for name, x in sums.items():
            err, size, plain, cut = (math.sqrt(y) for y in x)
            bound = u16 * size + 3 * plain + 2.0**-16 * cut + least * math.sqrt(sum(lens) * d)
            assert err <= bound, (name, h, err / size, plain / size, bound / size)


# ----------------------------------------------------------------- without the GPU's libraries


def test_the_package_imports_with_the_host_encoder_alone(tmp_path):
    """Without libmantis_hip.so and libmantis_torch.so the package imports and a model is built; a
    training operator raises, naming its library."""
    root = Path(mantisnet.__file__).resolve().parents[1]
    shutil.copytree(root / "mantisnet", tmp_path / "mantisnet", ignore=shutil.ignore_patterns("__pycache__"))
    shutil.copy(root / "libhexo_encoder.so", tmp_path)
    (tmp_path / "run.py").write_text(
        "import torch, mantisnet\n"
        "from mantisnet import ops\n"
        "mantisnet.MantisNet(mantisnet.MantisConfig())\n"
        "x, rng = torch.zeros(3, requires_grad=True), torch.zeros(2, dtype=torch.long)\n"
        "for f in (torch.ops.mantisnet.residual_dropout, ops.residual_dropout):\n"
        "    for y in (x, x.detach().to('meta')):\n"
        "        try:\n"
        "            f(y, None, rng.to(y.device), 0.5, 0)\n"
        "        except RuntimeError as err:\n"
        "            assert 'libmantis_torch.so' in str(err), err\n"
        "        else:\n"
        "            raise AssertionError('no error')\n"
        "print('done')\n")
    for broken in (False, True):  # not there; there, but not loadable
        if broken:
            (tmp_path / "libmantis_torch.so").write_bytes(b"no library")
        run = subprocess.run([sys.executable, str(tmp_path / "run.py")], capture_output=True, text=True, timeout=300)
        assert run.returncode == 0 and run.stdout.strip() == "done", run.stderr[-2000:]


# ----------------------------------------------------------------- the device's error words


_FIRST_USE = """
import sys, threading
import torch, mantisnet
from mantisnet import ops, tables
dev = torch.device("cuda:0")
x = torch.randn(40, device=dev)
offsets = torch.tensor([0, 40], device=dev)
bad = torch.tensor([[40]], device=dev)  # one past the run
torch.cuda.synchronize()

def call():
    return torch.ops.mantisnet.policy_log_probs(x, offsets, bad, 2)

def flagged():
    torch.cuda.synchronize()
    try:
        ops.raise_on_device_error()
    except ValueError:
        return True
    return False

def threads(first):
    gate = threading.Barrier(8)
    words = [None] * 8
    def work(i):
        with torch.cuda.stream(streams[i]):
            gate.wait()
            if i % 2 == first:
                call()
            else:
                words[i] = ops.error_flag(dev).data_ptr()
    streams = [torch.cuda.Stream() for _ in range(8)]
    all_ = [threading.Thread(target=work, args=(i,)) for i in range(8)]
    [t.start() for t in all_], [t.join() for t in all_]
    assert {w for w in words if w} == {ops.error_flag(dev).data_ptr()}

if sys.argv[1] == "threads":
    threads(0)
elif sys.argv[1] == "inference":
    with torch.inference_mode():
        call()
        ops.error_flag(dev)
else:
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call()
    assert not flagged()  # nothing has run yet
    for _ in range(3):
        graph.replay()
        assert flagged() and not flagged()
    graph.replay()
assert flagged() and not flagged()
call()
assert flagged() and not flagged()
print("done")
"""


@gpu
@pytest.mark.parametrize("first", ["threads", "inference", "capture"])
def test_error_words_are_there_before_anyone_writes_them(first):
    """The first use of a process, by several threads and streams, in inference mode or in a capture."""
    env = {**os.environ, "PYTHONPATH": str(Path(mantisnet.__file__).resolve().parents[1])}
    run = subprocess.run([sys.executable, "-c", _FIRST_USE, first], capture_output=True, text=True, timeout=100, env=env)
    assert run.returncode == 0 and run.stdout.strip().endswith("done"), run.stderr[-3000:]


@gpu
def test_threads_share_the_backward(device):
    """Eight threads, a stream and a variant each, against the same calls one by one."""
    cases = [base.relative_case([130, 64, 200][:1 + i % 3], 1 + i % 2, (16, 32, 64)[i % 3], (BF, HF)[i // 4], i,
                                device=device) for i in range(8)]
    want = [base._run_relative(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    gate, got = threading.Barrier(8), [None] * 8

    def work(i):
        with torch.cuda.stream(streams[i]):
            gate.wait()
            got[i] = [base._run_relative(cases[i]) for _ in range(5)]

    threads = [threading.Thread(target=work, args=(i,)) for i in range(8)]
    for x in threads:
        x.start()
    for x in threads:
        x.join()
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(one[n], w[n]) for one in g for n in w)


def test_forward_mode_is_refused():
    """A tangent is an error, with and without gradients asked for, not a zero."""
    import torch.autograd.forward_ad as fwad

    new = lambda *s, dtype=torch.float32: torch.empty(s, dtype=dtype, device="meta")  # noqa: E731
    i32, i64 = torch.int32, torch.int64
    q = new(2, 4, 9, 32, dtype=BF)
    rest = (new(4, 12), new(2, 9, 2, dtype=i32), new(5, 7, dtype=i32), new(2, dtype=i32), 4)
    rng = new(2, dtype=i64)
    calls = [
        (lambda x: OPS.fused_attention_relative(x, q, q, *rest)[0], q),
        (lambda x: OPS.fused_attention_relative(q, q, x, *rest)[0], q),
        (lambda x: OPS.fused_attention_relative(q, q, q, x, *rest[1:])[0], rest[0]),
        (lambda x: OPS.policy_log_probs(x, new(3, dtype=i64), new(2, 1, dtype=i64), 2)[0], new(10)),
        (lambda x: OPS.residual_dropout(x, None, rng, 0.5, 0), new(10)),
        (lambda x: OPS.residual_dropout(new(10), x, rng, 0.5, 0), new(10)),
    ]
    for call, x in calls:
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.func.jvp(call, (x,), (torch.empty_like(x),))
        with pytest.raises(RuntimeError):
            torch.func.jvp(lambda y: torch.func.grad(lambda z: call(z).sum())(y), (x,), (torch.empty_like(x),))
        for leaf in (x, x.clone().requires_grad_(True)):
            with fwad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
                call(fwad.make_dual(leaf, torch.empty_like(x)))
        call(x)


# ----------------------------------------------------------------- index tables that are none


@gpu
@pytest.mark.parametrize("n", [83, 30000])
@pytest.mark.parametrize("bad", [[0, 2.0, 0.5, 0.8], [0.2, 0.1, 0.6, 0.6], [-1.0, 0.5, 0.7, 0.9], [2.0, 3.0, 2.5, 1.5],
                                 [0.9, 0.1, 0.0, -1.0]])
def test_policy_gradients_outside_every_run_are_zero_whatever_the_offsets(device, n, bad):
    x = torch.randn(n, device=device, requires_grad=True)
    offsets = [int(f * n) for f in bad]
    moves = torch.full((3, 1), -1, device=device)
    entropy, lse = OPS.policy_log_probs(x, torch.tensor(offsets, device=device), moves, 2)[1:3]
    torch.full_like(x, math.nan)  # (its memory is the next result's)
    (dx,) = torch.autograd.grad(entropy.sum() + lse.sum(), x)
    with pytest.raises(ValueError, match="not ascending"):
        ops.raise_on_device_error(device)
    outside = torch.ones(n, dtype=torch.bool)
    for a, b in zip(offsets, offsets[1:]):
        if 0 <= a <= b <= n:
            outside[a:b] = False
    assert dx.isfinite().all() and not dx.cpu()[outside].any() and outside.any()


@gpu
@pytest.mark.parametrize("lens", [[70, 20], [200, 20], [150] * 60])
@pytest.mark.parametrize("bad", [math.nan, INF])
def test_relative_attention_a_bad_key_beside_lowest_scores(device, lens, bad):
    """A NaN (or infinite) score beside scores of the lowest finite value: its row is NaN, lse too."""
    q, k, v, bias, coords, buckets, sl, _n, _grad = base.relative_case(lens, 2, 32, BF, 9, n_latents=0, device=device)
    bias[:] = torch.finfo(torch.float32).min
    q = q.abs()
    k[0, 1, 5, 3] = bad
    out, lse, _ = OPS.fused_attention_relative(q, k, v, bias, coords, buckets, sl, 0)
    assert out[0, 1, :lens[0]].isnan().all()
    if math.isnan(bad):
        assert lse[0, 1, :lens[0]].isnan().all()
    assert not out[0, 0].isnan().any() and not lse[0, 0].isnan().any() and not out[1:].isnan().any()
    clean = lse[1, :, :lens[1]]
    assert torch.equal(clean, torch.full_like(clean, torch.finfo(torch.float32).min))


@gpu
def test_relative_attention_bias_gradient_of_long_rows(device):
    """dbias over 2,300 rows, most of whose pairs share a bucket: what stays of a row whose ds sum to
    zero is delta's own rounding.  In the 2-norm over four heads and four batches at most sqrt(5) times
    the fp32 formula's (summed up in float64): its roundings of scores, p and delta, and for each of the
    fp32 sums, delta's and the buckets' columns, those of its terms and of the sum, all independent."""
    n, heads, d = 2300, 4, 32
    buckets, count = tables.relative_buckets(12)
    err = low = 0.0
    for seed in range(4):
        q, k, v, _bias, coords, _b, lens, n_latents, grad = base.relative_case([n], heads, d, BF, seed, spread=26.0)
        bias = 0.5 * torch.randn(heads, count, generator=base._gen(seed))
        case = [x.to(device) for x in (q, k, v, bias, coords, buckets, lens)] + [n_latents, grad.to(device)]
        got = base._run_relative(tuple(case))["dbias"].double()
        pair = base._pairs(coords[0], buckets, n, n_latents, count).to(device)
        for h in range(heads):
            sums = []
            for dtype in (torch.float64, torch.float32):
                one = [x[0, h].to(device) for x in (q, k, v)] + [bias[h].to(device), pair, grad[0, h].to(device)]
                _, _, p, off = _elementwise(*one, dtype)
                sums.append(torch.bincount(pair.reshape(-1), (p * off).double().reshape(-1), minlength=count))
            err += float((got[h] - sums[0]).square().sum())
            low += float((sums[1] - sums[0]).square().sum())
    assert err <= 5 * low, math.sqrt(err / low)
