"""The expert-parallel layer: routing, dispatch, 4-bit products by expert and combine in a row, each step against a plain form of the
step in front of it, and the layer against the steps."""
import pytest
import torch

from helpers import run_ranks
from test_gpu_fp4 import check_gemm, gen, held, nearest, swiglu_reference

pytestmark = pytest.mark.gpu


def make(n, **kw):
    import hcomm_b200 as hb
    from hcomm_b200.parallel.ep import ExpertParallelMlp
    info = hb.get_root_info()
    comms = run_ranks(n, lambda r: (torch.cuda.set_device(0), hb.Communicator(n, info, r, buffer_mb=8))[1])
    layers = run_ranks(n, lambda r: (torch.cuda.set_device(0), ExpertParallelMlp(comms[r], **kw))[1])
    return comms, layers


def end(comms, layers):
    run_ranks(len(comms), lambda r: (torch.cuda.set_device(0), layers[r].destroy()))
    run_ranks(len(comms), lambda r: comms[r].destroy())


@pytest.mark.parametrize("tokens,experts,topk,hidden,inter,scoring", [(1, 8, 2, 512, 64, "softmax"), (50, 16, 4, 512, 160, "sigmoid"), (700, 8, 2, 1024, 512, "softmax")])
def test_each_step_of_one_rank(tokens, experts, topk, hidden, inter, scoring):
    from hcomm_b200.ops.fp4 import gemm_fp4, gemm_fp4_swiglu, quantize_fp4
    from hcomm_b200.ops.gemm import gemm_bf16
    from hcomm_b200.ops.moe import quantize_e4m3_1x128
    from hcomm_b200.ops.router import route
    g = gen(tokens)
    comms, (layer,) = make(1, experts=experts, topk=topk, hidden=hidden, intermediate=inter, max_tokens=tokens, scoring=scoring)
    try:
        x = torch.randn(tokens, hidden, device="cuda", generator=g).to(torch.bfloat16)
        valid = torch.rand(tokens, device="cuda", generator=g) < 0.9
        valid[0] = True
        out = layer(x, valid=valid).clone()
        r = layer.routing
        assert torch.equal(route(gemm_bf16(x, layer.router), topk, scoring=scoring, valid=valid).topk_idx, r.topk_idx)
        recv = layer.moe.dispatch(x, r.topk_idx)
        bounds, total = recv.expert_offsets.tolist(), recv.num_rows
        assert torch.equal(recv.expert_offsets.diff(), r.counts) and total == int(valid.sum()) * topk
        q, s = quantize_e4m3_1x128(x)
        tk = (recv.origin[:total] & 0xffffffff).long()
        rows = nearest(q.float() * s.repeat_interleave(128, 1))[tk // topk]
        h = gemm_fp4_swiglu(quantize_fp4(recv.rows, recv.scales, offsets=recv.expert_offsets), layer.gate, layer.up)
        y = gemm_fp4(quantize_fp4(h, offsets=recv.expert_offsets), layer.down)
        gate, up, down = held(layer.gate), held(layer.up), held(layer.down)
        for e, (lo, hi) in enumerate(zip(bounds, bounds[1:])):
            if lo < hi:
                want, tol = swiglu_reference(rows[lo:hi], gate[e], up[e])
                assert bool(((h[lo:hi].double() - want).abs() <= tol).all())
                check_gemm(y[lo:hi], nearest(h[lo:hi]), down[e])
        want = torch.zeros(tokens, hidden, dtype=torch.float64, device="cuda")
        terms = r.gates.double().view(-1)[tk].unsqueeze(1) * y[:total].double()
        want.index_add_(0, tk // topk, terms)
        size = torch.zeros_like(want).index_add_(0, tk // topk, terms.abs())
        # a rounding to bf16, and topk products and sums in 32 bits
        assert bool(((out.double() - want).abs() <= want.abs() * 2.0 ** -8 + size * topk * 2.0 ** -23).all())
        assert (out[~valid] == 0).all()
        # again, with the steps one by one, and in a graph: the same bits
        assert torch.equal(layer.moe.combine(y, r.gates), out)
        layer(x, out, valid)
        graph, into = torch.cuda.CUDAGraph(), torch.empty_like(out)
        with torch.cuda.graph(graph):
            layer(x, into, valid)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(into, out)
    finally:
        end(comms, [layer])


def test_batches_of_every_size_and_none():
    g = gen(5)
    comms, (layer,) = make(1, experts=16, topk=4, hidden=512, intermediate=96, max_tokens=200)
    try:
        x = torch.randn(200, 512, device="cuda", generator=g).to(torch.bfloat16)
        whole = layer(x).clone()
        for n in (200, 1, 33, 0, 128, 2):
            assert torch.equal(layer(x[:n]), whole[:n])
            assert int(layer.routing.counts.sum()) == 4 * n
        assert not layer(x, valid=torch.zeros(200, dtype=torch.bool, device="cuda")).any()
        assert layer.moe.overflow() == 0
        with pytest.raises(Exception):
            layer(torch.cat([x, x]))
    finally:
        end(comms, [layer])


def test_two_ranks_give_what_one_gives():
    from hcomm_b200.ops.fp4 import Fp4Tensor, quantize_fp4
    g = gen(77)
    experts, topk, hidden, inter, tokens = 16, 4, 512, 96, 40
    w = {name: (torch.randn(experts, *shape, device="cuda", generator=g) * 0.05).to(torch.bfloat16)
         for name, shape in (("w_gate", (inter, hidden)), ("w_up", (inter, hidden)), ("w_down", (hidden, inter)))}
    router = (torch.randn(experts, hidden, device="cuda", generator=g) * 0.05).to(torch.bfloat16)
    xs = [torch.randn(tokens, hidden, device="cuda", generator=g).to(torch.bfloat16) for _ in range(2)]
    options = dict(experts=experts, topk=topk, hidden=hidden, intermediate=inter, max_tokens=2 * tokens, w_router=router)
    comms, layers = make(1, **options, **w)
    want = layers[0](torch.cat(xs)).clone()
    torch.cuda.synchronize()
    end(comms, layers)
    import hcomm_b200 as hb
    from hcomm_b200.parallel.ep import ExpertParallelMlp
    info = hb.get_root_info()
    comms = run_ranks(2, lambda r: (torch.cuda.set_device(0), hb.Communicator(2, info, r, buffer_mb=8))[1])

    def layer(r):
        torch.cuda.set_device(0)
        mine = {name: v[r * 8:r * 8 + 8] for name, v in w.items()}
        if r == 1:                  # weights that are in 4 bits already
            mine = {name: quantize_fp4(v) for name, v in mine.items()}
            assert all(isinstance(v, Fp4Tensor) for v in mine.values())
        return ExpertParallelMlp(comms[r], **options, **mine)
    layers = run_ranks(2, layer)

    def step(r):
        torch.cuda.set_device(0)
        out = layers[r](xs[r])
        torch.cuda.synchronize()
        return out
    for _ in range(2):
        outs = run_ranks(2, step)
        assert torch.equal(torch.cat(outs), want)
    xs[1] = xs[1][:0]           # a rank without tokens; the other's go to the experts of both
    outs = run_ranks(2, step)
    assert torch.equal(outs[0], want[:tokens]) and outs[1].shape == (0, hidden)
    assert all(x.moe.overflow() == 0 for x in layers)
    end(comms, layers)


def test_refusals():
    import hcomm_b200 as hb
    from hcomm_b200.parallel.ep import ExpertParallelMlp
    torch.cuda.set_device(0)
    comm = hb.Communicator(1, hb.get_root_info(), 0, buffer_mb=4)
    for bad in (dict(experts=12), dict(w_gate=torch.zeros(8, 64, 256, device="cuda", dtype=torch.bfloat16)), dict(intermediate=48)):
        with pytest.raises(ValueError):
            ExpertParallelMlp(comm, **{**dict(experts=8, topk=2, hidden=512, intermediate=64, max_tokens=8), **bad})
    comm.destroy()


def _with_tokens_that_are_no_numbers(g, tokens, hidden):
    """x, which of its tokens are, and x without them."""
    x = torch.randn(tokens, hidden, device="cuda", generator=g).to(torch.bfloat16)
    bad = torch.zeros(tokens, dtype=torch.bool, device="cuda")
    bad[[0, 3, tokens - 2]] = True
    clean = x.clone()
    x[0, 5], x[3], x[tokens - 2, :2] = float("nan"), float("nan"), torch.tensor([float("inf"), float("-inf")], device="cuda")
    return x, bad, clean


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_a_token_that_is_no_number_comes_back_as_such(scoring):
    g = gen(91)
    comms, (layer,) = make(1, experts=16, topk=4, hidden=512, intermediate=96, max_tokens=70, scoring=scoring)
    try:
        x, bad, clean = _with_tokens_that_are_no_numbers(g, 70, 512)
        # weights of both signs: an infinite logit of each sign, or inf - inf; softmax knows neither, sigmoid not the latter
        layer.router.copy_(torch.randn(16, 512, device="cuda", generator=g).to(torch.bfloat16) * 0.02)
        layer.router[:, :2] = torch.tensor([[1.0, 1.0], [1.0, -1.0]], device="cuda").repeat(8, 1).to(torch.bfloat16)
        want = layer(clean).clone()
        out = layer(x).clone()
        assert torch.isnan(out[bad]).all() and torch.equal(out[~bad], want[~bad]) and not torch.isnan(want).any()
        # padding is not looked at, and the next batch does not know
        padded = layer(x, valid=~bad).clone()
        assert not padded[bad].any() and torch.equal(padded[~bad], want[~bad])
        assert torch.equal(layer(clean), want)
        graph, into = torch.cuda.CUDAGraph(), torch.empty_like(out)
        with torch.cuda.graph(graph):
            layer(x, into)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(into[~bad], want[~bad]) and torch.isnan(into[bad]).all()
    finally:
        end(comms, [layer])


def test_a_token_that_is_no_number_on_one_of_two_ranks():
    g = gen(92)
    comms, layers = make(2, experts=16, topk=4, hidden=512, intermediate=96, max_tokens=40)
    x, bad, clean = _with_tokens_that_are_no_numbers(g, 40, 512)

    def run(batches):
        def step(r):
            torch.cuda.set_device(0)
            out = layers[r](batches[r])
            torch.cuda.synchronize()
            return out.clone()
        return run_ranks(2, step)
    want, got = run([clean, clean]), run([x, clean])
    assert torch.isnan(got[0][bad]).all() and torch.equal(got[0][~bad], want[0][~bad]) and torch.equal(got[1], want[1])
    end(comms, layers)


@pytest.mark.parametrize("through_slots", [False, True])
def test_combine_carries_gates_that_are_no_numbers_where_it_is_asked_to(through_slots):
    import contextlib
    import hcomm_b200 as hb
    from hcomm_b200.ops.moe import MoeExchange
    g = gen(93)
    comm = hb.Communicator(1, hb.get_root_info(), 0, buffer_mb=4)
    moe = MoeExchange(comm, 8, 2, 512, 50)
    try:
        x = torch.randn(50, 512, device="cuda", generator=g).to(torch.bfloat16)
        idx = torch.randint(0, 8, (50, 2), device="cuda", generator=g, dtype=torch.int32)
        idx[::5] = -1
        idx[1::5, 1] = -1
        recv = moe.dispatch(x, idx)
        y = torch.randn(recv.num_rows + 50, 512, device="cuda", generator=g).to(torch.bfloat16)
        gates = torch.rand(50, 2, device="cuda", generator=g)
        gates[idx < 0] = 0
        want = moe.combine(y, gates).clone()
        gates[::5] = float("nan")
        gates[1::10, 1] = float("nan")
        bad = torch.isnan(gates).any(1)
        for mode in (contextlib.nullcontext(), torch.overrides.BaseTorchFunctionMode()):        # the native call, and the general one
            with mode:
                carried, left_out = y.clone(), y.clone()
                carried = moe.combine(carried, gates, carried[-50:] if through_slots else None, nan_gates=True)
                left_out = moe.combine(left_out, gates, left_out[-50:] if through_slots else None)
            assert torch.isnan(carried[bad]).all() and torch.equal(carried[~bad], want[~bad])
            assert torch.equal(left_out, want)          # as ever: a choice that was not sent adds nothing
    finally:
        moe.destroy()
        comm.destroy()


def test_a_result_with_more_rows_than_tokens():
    g = gen(95)
    comms, (layer,) = make(1, experts=8, topk=2, hidden=512, intermediate=64, max_tokens=20)
    try:
        x = torch.randn(20, 512, device="cuda", generator=g).to(torch.bfloat16)
        want = layer(x).clone()
        for n in (20, 7, 0):
            out = torch.full((20, 512), 5.0, device="cuda", dtype=torch.bfloat16)
            assert layer(x[:n], out) is out and torch.equal(out[:n], want[:n]) and (out[n:] == 5).all()
    finally:
        end(comms, [layer])
