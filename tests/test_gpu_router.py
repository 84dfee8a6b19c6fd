"""Routing, its counts, its balance loss and their gradients against a plain implementation in 64 bits.

Choices and counts are equal.  A score is an exponential divided by a sum of such: its argument is off by 2^-24 of the logits that go into
it (twice with a log-sigmoid, which is off by four roundings more), exp by 2^-23, each of the E / 32 + 5 additions, the
reciprocal and the products by 2^-24; `relative` adds these up.  Sums over tokens have positive terms, so their relative error is that of a
term plus a rounding for each addition in a row.  A gradient is a difference of such products: the bound is the relative
error of its terms times their magnitudes, three roundings more, and the rounding to its type."""
import contextlib

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SCALE, BALANCE = 2.5, 0.03


def gen(seed):
    torch.cuda.set_device(0)
    return torch.Generator(device="cuda").manual_seed(seed)


def reference(x, k, scoring, renormalize, bias=None, valid=None, idx=None):
    """idx, gates / SCALE, counts, tokens, p in 64 bits; the choice by sorting (expert, key) pairs in Python order."""
    x = x.double()
    t, e = x.shape
    if valid is not None:
        x = torch.where(valid.unsqueeze(1), x, -torch.inf)
    soft = scoring == "softmax"
    off = torch.isneginf(x)
    score = torch.exp(x - torch.nan_to_num(x.detach().amax(1, keepdim=True), neginf=0.0)) if soft else torch.where(off, 0.0, torch.sigmoid(x))
    if idx is None:
        key = (x if bias is None else score + bias.double()).detach().masked_fill(off, -torch.inf)
        idx = torch.tensor([[e_ if row[e_] > -float("inf") else -1 for e_ in sorted(range(e), key=lambda j: (-row[j], j))[:k]] for row in key.tolist()],
                           device=x.device).view(t, k)
    chosen = idx >= 0
    p = score / score.sum(1, keepdim=True).clamp_min(1e-300)
    share = torch.where(chosen, (p if soft else score).gather(1, idx.clamp_min(0)), 0.0)
    if renormalize:
        share = share / share.sum(1, keepdim=True).clamp_min(1e-300)
    counts = torch.bincount(idx[chosen], minlength=e)
    return idx, share, counts, t if valid is None else int(valid.sum()), p


def loss_of(counts, tokens, p, k):
    tokens = max(tokens, 1)
    return BALANCE * p.shape[1] * (counts.double() / (tokens * k) * p.sum(0) / tokens).sum()


def relative(x, e):
    big = float(x[torch.isfinite(x)].abs().max()) if torch.isfinite(x).any() else 0.0
    return 2.0 ** -24 * (e / 32 + 40 + 4 * big)


def gradient(x, idx, share, counts, tokens, p, scoring, renormalize, dgates, dloss, k):
    """By the formulas, and the magnitude of what is added up."""
    e = p.shape[1]
    tokens = max(tokens, 1)
    dg = torch.where(idx >= 0, SCALE * dgates.double(), 0.0)
    at = idx.clamp_min(0)
    u = (dloss * BALANCE * e * counts.double() / (tokens * k) / tokens).expand_as(p).clone()
    own, size = torch.zeros_like(p), torch.zeros_like(p)
    if renormalize:
        own.scatter_add_(1, at, share * (dg - (share * dg).sum(1, keepdim=True)))
        size.scatter_add_(1, at, share * (dg.abs() + (share * dg.abs()).sum(1, keepdim=True)))
    elif scoring == "softmax":
        u.scatter_add_(1, at, dg)
    else:
        own.scatter_add_(1, at, share * dg)
        size.scatter_add_(1, at, share * dg.abs())
    d = p * (u - (p * u).sum(1, keepdim=True)) + own
    size = size + p * (u.abs() + (p * u.abs()).sum(1, keepdim=True))
    if scoring == "sigmoid":
        back = torch.sigmoid(-x.double())
        d, size = torch.where(p + own.abs() > 0, d * back, 0.0), torch.where(p + own.abs() > 0, size * back, 0.0)
    return d, size


def make(g, t, e, dtype, masked):
    x = (1.5 * torch.randn(t, e, device="cuda", generator=g) + torch.randn(e, device="cuda", generator=g)).to(dtype)
    valid = None
    if masked:
        x[:, torch.rand(e, device="cuda", generator=g) < 0.2] = float("-inf")
        x[torch.rand(t, device="cuda", generator=g) < 0.1] = float("-inf")
        valid = torch.rand(t, device="cuda", generator=g) < 0.8
    return x, valid


CASES = [(1, 8, 2), (7, 1, 1), (33, 5, 5), (64, 60, 6), (300, 64, 6), (129, 100, 4), (500, 256, 8), (65, 300, 16), (40, 1000, 16), (70, 1024, 8), (9000, 16, 2)]


@pytest.mark.parametrize("t,e,k", CASES)
@pytest.mark.parametrize("scoring,renormalize,biased", [("softmax", True, False), ("softmax", False, False), ("sigmoid", True, True), ("sigmoid", False, False), ("sigmoid", True, False)])
@pytest.mark.parametrize("dtype,masked", [("fp32", True), ("bf16", False), ("fp16", True)])
def test_forward_and_backward(t, e, k, scoring, renormalize, biased, dtype, masked):
    from hcomm_b200.ops.router import route
    g = gen(t * e + k)
    x, valid = make(g, t, e, TYPES[dtype], masked)
    bias = torch.randn(e, device="cuda", generator=g) * 0.3 if biased else None
    idx, share, counts, tokens, p = reference(x, k, scoring, renormalize, bias, valid)
    rel = relative(x, e)
    x.requires_grad_()
    r = route(x, k, scoring=scoring, renormalize=renormalize, scale=SCALE, bias=bias, valid=valid, balance=BALANCE)
    assert torch.equal(r.topk_idx.long(), idx) and r.topk_idx.dtype == torch.int32
    assert torch.equal(r.counts.long(), counts)
    assert bool(((r.gates.double() - SCALE * share).abs() <= (rel + 2.0 ** -23) * SCALE * share + 1e-37).all())
    want = loss_of(counts, tokens, p, k)
    assert abs(r.loss.double() - want) <= want * (rel + 2.0 ** -24 * (t / 32 + 400 + e))
    # without a loss nothing else changes
    plain = route(x.detach(), k, scoring=scoring, renormalize=renormalize, scale=SCALE, bias=bias, valid=valid)
    assert plain.loss is None and torch.equal(plain.topk_idx, r.topk_idx) and torch.equal(plain.gates, r.gates) and torch.equal(plain.counts, r.counts)
    dgates, dloss = torch.randn(t, k, device="cuda", generator=g), torch.tensor(1.7 * t, device="cuda")
    (dx,) = torch.autograd.grad((r.gates, r.loss), x, (dgates, dloss))
    want, size = gradient(x.detach(), idx, share, counts, tokens, p, scoring, renormalize, dgates, dloss.double(), k)
    tol = (3 * rel + 2.0 ** -21) * size + torch.finfo(x.dtype).eps / 2 * want.abs() + (2.0 ** -25 if dtype == "fp16" else 1e-37)
    err = (dx.double() - want).abs()
    assert bool((err <= tol).all()), (err / tol).max().item()


@pytest.mark.parametrize("scoring,renormalize", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
def test_gradient_against_differences(scoring, renormalize):
    from hcomm_b200.ops.router import route
    g = gen(5)
    t, e, k = 24, 20, 3
    x, _ = make(g, t, e, torch.float32, False)
    dgates = torch.randn(t, k, device="cuda", generator=g)
    idx, share, counts, tokens, p = reference(x, k, scoring, renormalize)
    _, size = gradient(x, idx, share, counts, tokens, p, scoring, renormalize, dgates, torch.tensor(3.0, device="cuda", dtype=torch.float64), k)

    def value(x64):
        _, share, _, _, p = reference(x64, k, scoring, renormalize, idx=idx)
        return (SCALE * share * dgates.double()).sum() + 3.0 * loss_of(counts, tokens, p, k)
    x.requires_grad_()
    r = route(x, k, scoring=scoring, renormalize=renormalize, scale=SCALE, balance=BALANCE)
    ((r.gates * dgates).sum() + 3.0 * r.loss).backward()
    for _ in range(6):
        v = torch.randn(t, e, device="cuda", generator=g, dtype=torch.float64)
        h = 1e-5
        difference = (value(x.detach().double() + h * v) - value(x.detach().double() - h * v)) / (2 * h)
        # each entry of the gradient is off as in the test above; the difference by h^2 times a third derivative along v, below 10^4 here, and by
        # 2^-52 of values below 100 divided by h
        tol = ((3 * relative(x.detach(), e) + 2.0 ** -21 + 2.0 ** -24) * size * v.abs()).sum() + 1e-6 + 1e-8
        assert abs((x.grad.double() * v).sum() - difference) < tol


def test_gradients_of_one_output_alone():
    from hcomm_b200.ops.router import route
    g = gen(6)
    x, valid = make(g, 100, 64, torch.float32, True)
    x.requires_grad_()
    dgates = torch.randn(100, 6, device="cuda", generator=g)
    r = route(x, 6, valid=valid, balance=BALANCE)
    (both,) = torch.autograd.grad((r.gates, r.loss), x, (dgates, torch.ones((), device="cuda")), retain_graph=True)
    (gates,) = torch.autograd.grad(r.gates, x, dgates, retain_graph=True)
    (loss,) = torch.autograd.grad(r.loss, x, retain_graph=True)
    assert torch.allclose(gates + loss, both, rtol=1e-5, atol=1e-6)
    # broadcast gradients of the outputs, twice through the same graph, and no graph where none is asked for
    (a,) = torch.autograd.grad(r.gates.sum(), x, retain_graph=True)
    (b,) = torch.autograd.grad(r.gates, x, torch.ones_like(r.gates))
    assert torch.equal(a, b)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(r.gates.sum(), x)
    # logits that are themselves the result of something, used twice, changed in between
    y = x * 2
    a, c = route(y, 6, balance=BALANCE), route(y, 3)
    (d,) = torch.autograd.grad(a.gates.sum() + a.loss + c.gates.sum(), x)
    (e,), (f,) = (torch.autograd.grad(v, y) for v in (route(y, 6, balance=BALANCE).loss, route(y, 3, balance=BALANCE).gates.square().sum()))
    assert torch.isfinite(d).all() and torch.allclose(d, 2 * e, rtol=1e-4, atol=1e-6) and f.abs().sum() > 0       # gates of a token add up to 1
    r = route(y, 6)
    y.detach().mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(r.gates.sum(), x)
    with torch.no_grad():
        assert not route(x, 6, balance=BALANCE).gates.requires_grad
    assert not r.topk_idx.requires_grad and not r.counts.requires_grad
    bf = x.detach().to(torch.bfloat16).requires_grad_()
    with pytest.raises(RuntimeError):
        y = route(bf, 6)
        (grad,) = torch.autograd.grad(y.gates, bf, dgates, create_graph=True)
        grad.sum().backward()


def test_ties_go_to_the_lowest_expert():
    from hcomm_b200.ops.router import route
    torch.cuda.set_device(0)
    for e in (8, 64, 100, 256, 1024):
        for value in (0.0, 3.5, torch.finfo(torch.float32).min, -1e30):
            r = route(torch.full((3, e), value, device="cuda"), 4)
            assert r.topk_idx.tolist() == [[0, 1, 2, 3]] * 3
            assert torch.allclose(r.gates, torch.full_like(r.gates, 0.25))
        zeros = torch.zeros(1, e, device="cuda")
        zeros[0, ::2] = -0.0
        assert route(zeros, 4).topk_idx.tolist() == [[0, 1, 2, 3]]
        x = torch.zeros(2, e, device="cuda", dtype=torch.bfloat16)
        x[0, e - 1] = x[0, e // 2] = 1
        x[1, 1] = float("inf")
        assert route(x[:1], 3).topk_idx.tolist() == [[e // 2, e - 1, 0]]
        r = route(x[1:], 3, scoring="sigmoid", bias=torch.zeros(e, device="cuda"))
        assert r.topk_idx.tolist() == [[1, 0, 2]] and torch.allclose(r.gates, torch.tensor([[0.5, 0.25, 0.25]], device="cuda"))
    lowest = torch.full((1, 64), float("-inf"), device="cuda", dtype=torch.bfloat16)
    lowest[0, 5], lowest[0, 60] = torch.finfo(torch.bfloat16).min, 2.0
    r = route(lowest, 4)
    assert r.topk_idx.tolist() == [[60, 5, -1, -1]] and r.gates.tolist() == [[1, 0, 0, 0]]


def test_scores_that_32_bits_cannot_tell_apart():
    from hcomm_b200.ops.router import route
    torch.cuda.set_device(0)
    # sigmoids of 20 and more differ from 1 by less than half a step of 32 bits; the larger one is chosen all the same
    x = torch.arange(20, 36, device="cuda", dtype=torch.float32).view(1, 16)
    assert route(x, 3, scoring="sigmoid", bias=torch.zeros(16, device="cuda")).topk_idx.tolist() == [[15, 14, 13]]
    bias = torch.zeros(16, device="cuda")
    bias[0], bias[15] = 1e-8, float("-inf")
    assert route(x, 3, scoring="sigmoid", bias=bias).topk_idx.tolist() == [[0, 14, 13]]
    # far down, sigmoids that 32 bits round to nothing still have shares
    r = route(torch.tensor([[-200.0, -201.0, -300.0]], device="cuda"), 2, scoring="sigmoid")
    want = torch.softmax(torch.tensor([0.0, -1.0], dtype=torch.float64), 0)
    assert torch.allclose(r.gates.double().cpu(), want, rtol=1e-5)


def test_rows_that_are_no_numbers():
    from hcomm_b200.ops.router import route
    g = gen(9)
    for scoring, renormalize in (("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)):
        x, _ = make(g, 50, 64, torch.float32, False)
        clean = route(x, 4, scoring=scoring, renormalize=renormalize)
        x[7, 3] = float("nan")
        x[9, 60] = float("inf") if scoring == "softmax" else float("nan")
        x.requires_grad_()
        r = route(x, 4, scoring=scoring, renormalize=renormalize, balance=BALANCE)
        good = torch.ones(50, dtype=torch.bool, device="cuda")
        good[[7, 9]] = False
        assert (r.topk_idx[~good] == -1).all() and torch.isnan(r.gates[~good]).all() and torch.isnan(r.loss)
        assert torch.equal(r.topk_idx[good], clean.topk_idx[good]) and torch.equal(r.gates[good], clean.gates[good])
        assert int(r.counts.sum()) == 48 * 4
        (d,) = torch.autograd.grad(r.gates, x, torch.ones_like(r.gates))
        assert torch.isnan(d[~good]).all() and torch.isfinite(d[good]).all()
        # in padding they are not looked at
        r = route(x, 4, scoring=scoring, renormalize=renormalize, balance=BALANCE, valid=good)
        assert torch.isfinite(r.loss) and (r.gates[~good] == 0).all()
        (d,) = torch.autograd.grad(r.loss, x)
        assert (d[~good] == 0).all() and torch.isfinite(d).all()


def test_strides_alignment_empty_and_masked_batches():
    from hcomm_b200.ops.router import route
    g = gen(12)
    for dtype in TYPES.values():
        big, _ = make(g, 61, 300, dtype, False)
        for view in (big[:, 1:257], big[:, 8:264], big[::2, :64], big[:1, :60], big.view(-1)[3:3 + 60 * 300].view(60, 300)[:, :128]):
            base = view.contiguous()
            r, want = route(view, 4, balance=BALANCE), route(base, 4, balance=BALANCE)
            for a, b in zip(r, want):
                assert torch.equal(a, b)
            leaf, other = view.detach().requires_grad_(), base.detach().requires_grad_()
            (d,), (dw,) = (torch.autograd.grad(route(v, 4, balance=BALANCE).loss, v) for v in (leaf, other))
            assert torch.equal(d, dw)
    x = torch.empty(0, 64, device="cuda", requires_grad=True)
    r = route(x, 4, balance=BALANCE)
    assert r.topk_idx.shape == (0, 4) and int(r.counts.sum()) == 0 and r.loss == 0
    (d,) = torch.autograd.grad(r.loss, x)
    assert d.shape == x.shape
    x, _ = make(g, 100, 64, torch.float32, False)
    x.requires_grad_()
    for bad in (dict(valid=torch.zeros(100, dtype=torch.bool, device="cuda")), dict()):
        y = x if bad else torch.full_like(x, float("-inf")).requires_grad_()
        r = route(y, 4, balance=BALANCE, **bad)
        assert (r.topk_idx == -1).all() and (r.gates == 0).all() and r.loss == 0 and int(r.counts.sum()) == 0
        (d,) = torch.autograd.grad((r.gates, r.loss), y, (torch.ones_like(r.gates), torch.ones((), device="cuda")))
        assert (d == 0).all()


def test_same_bits_every_time_and_in_a_replayed_graph():
    from hcomm_b200.ops.router import route
    g = gen(15)
    x, valid = make(g, 20000, 128, torch.bfloat16, True)
    x.requires_grad_()
    ones = torch.ones((), device="cuda")

    def step():
        r = route(x, 4, valid=valid, balance=BALANCE)
        return *r, torch.autograd.grad((r.gates, r.loss), x, (torch.ones_like(r.gates), ones))[0]
    first = [t.detach().clone() for t in step()]
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(step(), first))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = step()
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, first))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept = [t.detach() for t in step()]
        graphs.append((graph, kept))
    with torch.no_grad():
        x.copy_(make(g, 20000, 128, torch.bfloat16, False)[0])
    want = [t.detach().clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(4):          # two graphs at the same time
        graphs[0][0].replay()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
    torch.cuda.synchronize()
    for _, kept in graphs:
        assert all(torch.equal(a, b) for a, b in zip(kept, want))


def test_sums_over_a_communicator():
    import hcomm_b200 as hb
    from hcomm_b200.ops.router import route
    g = gen(18)
    comm = hb.Communicator(1, hb.get_root_info(), 0, buffer_mb=4)
    try:
        for t in (20, 3000):
            x, valid = make(g, t, 64, torch.float32, True)
            x.requires_grad_()
            alone, shared = (route(x, 6, valid=valid, balance=BALANCE, comm=c) for c in (None, comm))
            assert torch.equal(alone.counts, shared.counts) and torch.equal(alone.gates, shared.gates)
            assert torch.allclose(alone.loss, shared.loss, rtol=1e-6)
            (a,), (b,) = (torch.autograd.grad(r.loss, x) for r in (alone, shared))
            assert torch.equal(a, b)
            assert torch.equal(route(x.detach(), 6, comm=comm).topk_idx, route(x.detach(), 6).topk_idx)
    finally:
        comm.destroy()


def test_threads_whose_calls_are_the_first():
    import subprocess
    import sys
    from pathlib import Path
    program = """
import sys, threading
sys.path.insert(0, {root!r})
import torch
from hcomm_b200.ops.router import route
x = torch.randn(40, 64, device="cuda")
got, bad = [], []
def work():
    try:
        got.append(route(x, 4).topk_idx)
    except BaseException as e:
        bad.append(e)
threads = [threading.Thread(target=work) for _ in range(16)]
for t in threads: t.start()
for t in threads: t.join()
torch.cuda.synchronize()
print(len(got), bad, all(torch.equal(g, got[0]) for g in got))
""".format(root=str(Path(__file__).resolve().parent.parent))
    res = subprocess.run([sys.executable, "-c", program], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and res.stdout.split() == ["16", "[]", "True"], res.stdout + res.stderr


def test_refusals():
    import numpy as np
    from hcomm_b200.ops.router import route
    torch.cuda.set_device(0)
    x = torch.zeros(4, 8, device="cuda")
    assert torch.equal(route(x, np.int64(3)).topk_idx, route(x, 3).topk_idx)
    with pytest.raises(TypeError):
        route(x, 2.0)
    for error, args, kw in ((ValueError, (x, 9), {}), (ValueError, (x, 0), {}), (ValueError, (x, 2), dict(scoring="tanh")), (TypeError, (x.long(), 2), {}), (TypeError, (x[0], 2), {}),
                            (ValueError, (x.t(), 2), {}), (ValueError, (x.cpu(), 2), {}), (ValueError, (torch.zeros(2, 1025, device="cuda"), 2), {}),
                            (ValueError, (torch.zeros(2, 64, device="cuda"), 17), {}), (ValueError, (x, 2), dict(bias=torch.zeros(8, device="cuda"))),
                            (ValueError, (x, 2), dict(scoring="sigmoid", bias=torch.zeros(7, device="cuda"))), (ValueError, (x, 2), dict(scoring="sigmoid", bias=torch.zeros(8))),
                            (ValueError, (x, 2), dict(valid=torch.zeros(3, dtype=torch.bool, device="cuda"))), (ValueError, (x, 2), dict(valid=torch.zeros(4, device="cuda"))),
                            (ValueError, (torch.zeros(1, 8, device="cuda").expand(4, 8), 2), {}), (TypeError, (x.double(), 2), {})):
        with pytest.raises(error):
            route(*args, **kw)


@pytest.mark.parametrize("topk", [2 ** 32 + 2, 2 ** 64 + 2, -2 ** 32 + 2])
def test_choices_beyond_32_bits_are_refused(topk):
    from hcomm_b200.ops.router import route
    with pytest.raises(ValueError):
        route(torch.zeros(4, 8, device="cuda"), topk)


def test_a_coefficient_that_is_0_in_32_bits_makes_a_loss_of_0():
    from hcomm_b200.ops.router import route
    x = torch.randn(4, 8, device="cuda", requires_grad=True)
    for mode in (contextlib.nullcontext(), torch.overrides.BaseTorchFunctionMode()):        # the native call, and the general one
        with mode:
            loss = route(x, 2, balance=1e-50).loss
        assert loss is not None and loss.item() == 0
        assert torch.equal(torch.autograd.grad(loss, x)[0], torch.zeros_like(x))


@pytest.mark.parametrize("e,k", [(64, 6), (256, 8), (1024, 16)])
def test_gradients_of_tokens_that_share_experts_in_turn(e, k):
    """A warp's tokens, one after the other, choose the same experts by other lanes: what one leaves in the row that they share is not the next one's."""
    from hcomm_b200.ops.router import route
    g = gen(e)
    t = 148 * 2 * 32 * 3 + 5
    order = torch.stack([torch.randperm(k, device="cuda", generator=g) for _ in range(16)])[torch.arange(t, device="cuda") // 32 % 16]
    x = torch.randn(t, e, device="cuda", generator=g) * 0.1
    x[:, ::e // k] = 0
    x.scatter_(1, torch.arange(k, device="cuda") * (e // k) + torch.zeros_like(order), 3.0 + order * 0.25)
    x.requires_grad_()
    dgates = torch.randn(t, k, device="cuda", generator=g)
    r = route(x, k, scale=SCALE)
    share = torch.softmax(x.detach().double().gather(1, r.topk_idx.long()), 1)
    none = torch.zeros((), device="cuda", dtype=torch.float64)
    want, size = gradient(x.detach(), r.topk_idx.long(), share, torch.zeros(e, device="cuda"), t, torch.zeros_like(x, dtype=torch.float64), "softmax", True, dgates, none, k)
    tol = (3 * relative(x.detach(), e) + 2.0 ** -21 + 2.0 ** -24) * size + 1e-37
    for _ in range(3):
        (dx,) = torch.autograd.grad(r.gates, x, dgates, retain_graph=True)
        assert bool(((dx.double() - want).abs() <= tol).all())


def test_threads_whose_calls_need_different_shared_memory():
    """Both sizes run the same kernel with more than 48 KB of shared memory; neither may lower what the other one is allowed."""
    import threading
    from hcomm_b200.ops.router import route
    g = gen(33)
    xs = [torch.randn(64, e, device="cuda", generator=g) for e in (800, 1024)]
    want = [route(x, 8, balance=BALANCE) for x in xs]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        torch.cuda.set_device(0)
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(3000):
                    r = route(xs[i], 8, balance=BALANCE)
                if not torch.equal(r.topk_idx, want[i].topk_idx) or not torch.equal(r.loss, want[i].loss):
                    bad.append(i)
        except RuntimeError as e:
            bad.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1, 0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


@pytest.mark.parametrize("requires_grad", [False, True])
def test_a_tangent_is_refused_and_not_dropped(requires_grad):
    import torch.autograd.forward_ad as fwad
    from hcomm_b200.ops.router import route
    x = torch.randn(6, 8, device="cuda", requires_grad=requires_grad)
    with fwad.dual_level():
        dual = fwad.make_dual(x, torch.ones_like(x))
        for mode in (contextlib.nullcontext(), torch.overrides.BaseTorchFunctionMode(), torch.no_grad()):        # the native call, the general one, without reverse mode
            with mode, pytest.raises(RuntimeError, match="jvp"):
                route(dual, 2, balance=BALANCE)
        assert route(x, 2).topk_idx.shape == (6, 2)         # no tangent, no refusal
    assert torch.equal(route(dual, 2).topk_idx, route(x, 2).topk_idx)


def test_saved_tensors_pass_hooks_and_checkpoints():
    """What the gradient needs is saved as any operator's is: hooks may keep it elsewhere, a checkpoint may make it again."""
    from torch.utils.checkpoint import checkpoint
    from hcomm_b200.ops.router import route
    g = gen(44)
    wide, valid = make(g, 300, 96, torch.bfloat16, True)
    x = wide[:, :64].detach().requires_grad_()
    dgates = torch.randn(300, 6, device="cuda", generator=g)

    def loss(v):
        r = route(v * 1.5, 6, valid=valid, balance=BALANCE)
        return (r.gates * dgates).sum() + 7 * r.loss
    (want,) = torch.autograd.grad(loss(x), x)
    assert want.abs().sum() > 0
    for mode in (contextlib.nullcontext(), torch.overrides.BaseTorchFunctionMode()):
        with mode:
            packed = []
            with torch.autograd.graph.saved_tensors_hooks(lambda t: packed.append(t.shape) or t.cpu(), lambda t: t.cuda()):
                kept = loss(x)
            assert packed.count((300, 64)) >= 1 and packed.count((300, 6)) >= 1
            assert torch.equal(torch.autograd.grad(kept, x)[0], want)
            with torch.autograd.graph.save_on_cpu():
                kept = loss(x)
            assert torch.equal(torch.autograd.grad(kept, x)[0], want)
            for reentrant in (False, True):
                y = x.detach().requires_grad_()
                checkpoint(loss, y, use_reentrant=reentrant).backward()
                assert torch.equal(y.grad, want)


@pytest.mark.parametrize("scoring,renormalize", [("softmax", True), ("softmax", False), ("sigmoid", True)])
@pytest.mark.parametrize("sizes", [(40, 3000), (3000, 0), (1, 33)])
def test_one_loss_of_two_ranks(sizes, scoring, renormalize):
    """Counts and loss are those of both ranks' tokens, and each rank's gradient is that of the one loss."""
    import hcomm_b200 as hb
    from hcomm_b200.ops.router import route
    from helpers import run_ranks
    g = gen(sum(sizes))
    e, k = 64, 6
    x, valid = make(g, sum(sizes), e, torch.float32, True)
    dgates, dloss = torch.randn(sum(sizes), k, device="cuda", generator=g), torch.tensor(1.3 * sum(sizes), device="cuda")
    idx, share, counts, tokens, p = reference(x, k, scoring, renormalize, None, valid)
    rel = relative(x, e)
    want = loss_of(counts, tokens, p, k)
    want_dx, size = gradient(x, idx, share, counts, tokens, p, scoring, renormalize, dgates, dloss.double(), k)
    tol = (3 * rel + 2.0 ** -21 + 2.0 ** -24) * size + 1e-37
    spans = (slice(0, sizes[0]), slice(sizes[0], sum(sizes)))
    info = hb.get_root_info()
    comms = run_ranks(2, lambda r: (torch.cuda.set_device(0), hb.Communicator(2, info, r, buffer_mb=4))[1])
    torch.cuda.synchronize()

    def step(r):
        torch.cuda.set_device(0)
        mine = x[spans[r]].clone().requires_grad_()
        out = route(mine, k, scoring=scoring, renormalize=renormalize, scale=SCALE, valid=valid[spans[r]], balance=BALANCE, comm=comms[r])
        (dx,) = torch.autograd.grad((out.gates, out.loss), mine, (dgates[spans[r]], dloss))
        without = route(mine.detach(), k, scoring=scoring, renormalize=renormalize, scale=SCALE, valid=valid[spans[r]], comm=comms[r])
        torch.cuda.synchronize()
        assert without.loss is None and torch.equal(without.counts, out.counts) and torch.equal(without.topk_idx, out.topk_idx)
        return out, dx
    for _ in range(2):
        got = run_ranks(2, step)
        for r, (out, dx) in enumerate(got):
            assert torch.equal(out.topk_idx.long(), idx[spans[r]]) and torch.equal(out.counts.long(), counts)
            assert abs(out.loss.double() - want) <= want * (rel + 2.0 ** -24 * (sum(sizes) / 32 + 401 + e))
            assert bool(((dx.double() - want_dx[spans[r]]).abs() <= tol[spans[r]]).all())
        assert torch.equal(got[0][0].loss, got[1][0].loss)
    run_ranks(2, lambda r: comms[r].destroy())
