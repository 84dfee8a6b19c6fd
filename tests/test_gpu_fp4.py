"""Microscaled 4-bit quantisation and products against plain implementations in 64 bits.

Quantisation is exact arithmetic followed by one rounding to the nearest of sixteen values, so it is compared for equality.  A product
is off by one rounding to bf16 (2^-8 of the value) and by its fp32 sums: K terms, each addition off by at most 2^-23 of what was added up so
far (the tensor core may cut off instead of rounding), so by less than K 2^-23 sum |a b|."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def nearest(x):
    """fp64 values of x [..., cols] in blocks of 32, each to the nearest of the sixteen by a search over all of them."""
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=x.device)
    even = torch.tensor([0, 2, 4, 6], device=x.device)
    blocks = x.double().reshape(-1, 32)
    amax = blocks.abs().amax(1)
    _, e = torch.frexp(torch.where(torch.isfinite(amax), amax, 1.0))
    power = torch.where(amax > 0, (e - 3).clamp(-127, 127), -127)
    unit = torch.ldexp(torch.ones_like(amax), power).unsqueeze(1)
    a = (blocks.abs() / unit).clamp_max(6.0)
    d = (a.unsqueeze(-1) - grid).abs()
    d[..., even] -= 1e-9            # of two that are as near the one with an even code; other distances differ by 2^-22 and more
    q = grid[d.argmin(-1)] * blocks.sign() * unit
    q[~torch.isfinite(amax)] = float("nan")
    return q.view(x.shape)


def held(q):
    """fp64 values of an Fp4Tensor without groups, read from its bytes."""
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=q.device)
    grid = torch.cat([grid, -grid])
    codes = torch.stack([q.values & 15, q.values >> 4], -1).flatten(-2)
    s = q.block_scales()
    unit = torch.ldexp(torch.ones(s.shape, dtype=torch.float64, device=s.device), s.int() - 127)
    unit[s == 255] = float("nan")
    return grid[codes.long()] * unit.repeat_interleave(32, -1)


def same(a, b):
    return torch.equal(torch.nan_to_num(a.double(), nan=1e30), torch.nan_to_num(b.double(), nan=1e30))


def gen(seed):
    torch.cuda.set_device(0)
    return torch.Generator(device="cuda").manual_seed(seed)


def spread(g, *shape):
    """Values whose magnitudes span many powers of two from block to block."""
    x = torch.randn(*shape, device="cuda", generator=g)
    return x * torch.exp2(torch.randint(-12, 12, (*shape[:-1], shape[-1] // 32), device="cuda", generator=g).float()).repeat_interleave(32, -1)


def weights(g, *shape):
    from hcomm_b200.ops.fp4 import Fp4Tensor
    codes = torch.randint(0, 256, (*shape[:-1], shape[-1] // 2), device="cuda", generator=g, dtype=torch.uint8)
    return Fp4Tensor.from_parts(codes, torch.randint(120, 132, (*shape[:-1], shape[-1] // 32), device="cuda", generator=g, dtype=torch.uint8))


def bound(a, b, want):
    return want.abs() * 2.0 ** -8 + a.shape[1] * 2.0 ** -23 * (a.abs() @ b.abs().t()) + 1e-38


def check_gemm(out, a, b):
    want = a @ b.t()
    err = (out.double() - want).abs()
    tol = bound(a, b, want)
    assert bool((err <= tol).all()), (err / tol).max().item()


def swiglu_reference(a, g, u):
    """The value and how far its fp32 form, rounded to bf16, may be off."""
    gate, up = a @ g.t(), a @ u.t()
    eg, eu = (a.shape[1] * 2.0 ** -23 * (a.abs() @ w.abs().t()) for w in (g, u))
    silu = gate * torch.sigmoid(gate)
    # |silu'| < 1.1; exp, sum, quotient and product are off by less than 2^-20 together, exp by |g| 2^-22 more (its argument is rounded)
    eg = 1.1 * eg + silu.abs() * (2.0 ** -20 + gate.abs() * 2.0 ** -22)
    want = silu * up
    return want, want.abs() * 2.0 ** -8 + eg * (up.abs() + eu) + silu.abs() * eu + 1e-38


@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 96), (128, 128), (130, 416), (257, 1024), (16, 28672), (1000, 2080)])
@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_quantise_and_back(rows, cols, dtype):
    from hcomm_b200.ops.fp4 import dequantize_fp4, quantize_fp4
    x = spread(gen(rows + cols), rows, cols).to(TYPES[dtype])
    x[0, :32] = 0
    q = quantize_fp4(x)
    want = nearest(x)
    assert same(held(q), want)
    assert same(dequantize_fp4(q), want)
    assert same(dequantize_fp4(q, torch.float32), want)
    tiles = q.scales.view(-1, -(-cols // 128), 32, 4, 4)[:, -1]
    assert cols % 128 == 0 or not tiles[:rows // 128, :, :, cols % 128 // 32:].any()         # bytes behind the last column


def test_ties_borders_and_values_that_are_no_numbers():
    from hcomm_b200.ops.fp4 import dequantize_fp4, quantize_fp4
    torch.cuda.set_device(0)
    half = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 7.99, 4.0, 0.2499, 0.2501, 4.9999, 5.0001, 6.0, 0.0], device="cuda")
    row = torch.cat([half, -half])
    x = torch.stack([row * 2.0 ** p for p in (-140, -130, -126, -100, -1, 0, 1, 100, 125)])
    x = torch.cat([x, torch.full((6, 32), 1.0, device="cuda")])
    x[9, 3], x[10, 5], x[11, 31], x[12], x[13], x[14] = float("nan"), float("inf"), float("-inf"), 1e-45, torch.finfo(torch.float32).max, -0.0
    want = nearest(x)
    q = quantize_fp4(x)
    assert same(held(q), want) and same(dequantize_fp4(q, torch.float32), want)
    assert torch.isnan(want[9:12]).all() and not torch.isnan(want[12:]).any()
    low = torch.full((2, 64), torch.finfo(torch.bfloat16).min, device="cuda", dtype=torch.bfloat16)
    assert same(held(quantize_fp4(low)), nearest(low))


def test_strides_alignment_and_several_matrices():
    from hcomm_b200.ops.fp4 import dequantize_fp4, quantize_fp4
    g = gen(3)
    for dtype in TYPES.values():
        big = spread(g, 40, 512).to(dtype)
        for x in (big[:, 32:288], big[::3, :256], big.view(-1)[1:1 + 39 * 512].view(39, 512)[:, :96], big[:, 3:67], big[:1, :64]):
            assert same(held(quantize_fp4(x)), nearest(x))
        cube = spread(g, 5, 130, 160).to(dtype)
        for x in (cube, cube[::2], cube[:, 1:, :96], cube.transpose(0, 1), cube[:1]):
            q = quantize_fp4(x)
            assert same(held(q), nearest(x)) and same(dequantize_fp4(q, torch.float32), nearest(x))
    row = spread(g, 1, 96)
    assert same(held(quantize_fp4(row.expand(70, 96))), nearest(row).expand(70, 96))
    for shape in ((0, 64), (4, 0), (0, 3, 32), (2, 0, 32)):
        q = quantize_fp4(torch.empty(shape, device="cuda"))
        assert q.shape == shape and dequantize_fp4(q).shape == shape


@pytest.mark.parametrize("rows,cols,split", [(300, 256, [0, 0, 130, 130, 258, 290]), (5, 128, [0, 5]), (600, 640, [0, 1, 2, 130, 600]), (64, 128, [0] * 9), (40, 256, [8, 20, 33]),
                                             (2000, 128, list(range(0, 2000, 2)))])
def test_rows_grouped_by_expert(rows, cols, split):
    from hcomm_b200.ops.fp4 import Fp4Tensor, dequantize_fp4, quantize_fp4
    g = gen(rows)
    x = spread(g, rows, cols).to(torch.bfloat16)
    offsets = torch.tensor(split, device="cuda", dtype=torch.int32)
    q = quantize_fp4(x, offsets=offsets)
    lo, hi = split[0], split[-1]
    assert same(dequantize_fp4(q, torch.float32)[lo:hi], nearest(x)[lo:hi])
    # each expert's tiles are those of its rows alone
    tile = 0
    for a, b in zip(split, split[1:]):
        if a == b:
            continue
        alone = quantize_fp4(x[a:b].contiguous())
        n = -(-(b - a) // 128) * -(-cols // 128)
        mine = Fp4Tensor(q.values[a:b], q.scales[tile:tile + n])
        assert torch.equal(mine.block_scales(), alone.block_scales()) and torch.equal(mine.values, alone.values)
        tile += n
    assert tile <= q.scales.shape[0]


def test_offsets_that_leave_the_rows_touch_nothing_else():
    from hcomm_b200.ops.fp4 import gemm_fp4, quantize_fp4
    g = gen(8)
    x, w = spread(g, 200, 256), weights(g, 4, 136, 256)
    for split in ([0, 50, 500, 500, 500], [-7, 20, 10, 60, 150], [200, 100, 50, 20, 0]):
        clean, top = [], 0
        for v in split:
            top = max(top, min(max(v, 0), 200))
            clean.append(top)
        out = torch.full((200, 136), 7.0, device="cuda", dtype=torch.bfloat16)
        q = quantize_fp4(x, offsets=torch.tensor(split, device="cuda", dtype=torch.int32))
        gemm_fp4(q, w, out)
        for e, (a, b) in enumerate(zip(clean, clean[1:])):
            if a < b:
                check_gemm(out[a:b], nearest(x[a:b]), held(w)[e])
        assert (out[:clean[0]] == 7).all() and (out[clean[-1]:] == 7).all()


def test_rows_as_the_exchange_delivers_them():
    from hcomm_b200.ops.fp4 import dequantize_fp4, quantize_fp4
    from hcomm_b200.ops.moe import quantize_e4m3_1x128
    g = gen(11)
    rows, scales = quantize_e4m3_1x128(spread(g, 150, 512))
    want = nearest(rows.float() * scales.repeat_interleave(128, 1))
    assert same(held(quantize_fp4(rows, scales)), want)
    offsets = torch.tensor([0, 3, 3, 140], device="cuda", dtype=torch.int32)
    assert same(dequantize_fp4(quantize_fp4(rows, scales, offsets=offsets), torch.float32)[:140], want[:140])
    wide = torch.cat([scales, scales], 1)
    assert same(held(quantize_fp4(rows[:, :256], wide[:, :2])), want[:, :256])


@pytest.mark.parametrize("m,n,k", [(1, 8, 32), (1, 1, 96), (16, 136, 96), (33, 100, 64), (127, 257, 160), (128, 128, 256), (129, 384, 1024), (300, 1000, 2080), (64, 4096, 512),
                                   (1000, 8, 288), (2500, 3584, 416), (2048, 4096, 320), (4100, 1030, 256)])
def test_product(m, n, k):
    from hcomm_b200.ops.fp4 import gemm_fp4, quantize_fp4, take_kernel_error
    g = gen(m + n + k)
    a, b = quantize_fp4(spread(g, m, k)), weights(g, n, k)
    out = gemm_fp4(a, b)
    torch.cuda.synchronize()
    assert take_kernel_error() == 0
    check_gemm(out, held(a), held(b))


@pytest.mark.parametrize("m,n,k", [(1, 8, 32), (5, 100, 96), (130, 128, 256), (300, 1000, 512), (1111, 4096, 320)])
def test_gated_product(m, n, k):
    from hcomm_b200.ops.fp4 import gemm_fp4_swiglu, quantize_fp4
    g = gen(m + n + k)
    a = quantize_fp4(torch.randn(m, k, device="cuda", generator=g))
    gate, up = quantize_fp4(torch.randn(n, k, device="cuda", generator=g) * 0.2), weights(g, n, k)
    out = gemm_fp4_swiglu(a, gate, up)
    want, tol = swiglu_reference(held(a), held(gate), held(up))
    err = (out.double() - want).abs()
    assert bool((err <= tol).all()), (err / tol).max().item()


@pytest.mark.parametrize("rows,n,k,split", [(64, 136, 96, [0, 0, 10, 10, 50]), (700, 384, 256, [0, 129, 129, 400, 656, 700]), (300, 100, 160, [20, 21, 300]), (8, 256, 128, [0] * 33),
                                            (1, 64, 32, [0, 0, 1]), (5000, 1024, 192, [0, 2000, 2001, 5000]), (2000, 40, 64, list(range(0, 2000, 2)))])
@pytest.mark.parametrize("gated", [False, True])
def test_products_by_expert(rows, n, k, split, gated):
    from hcomm_b200.ops.fp4 import gemm_fp4, gemm_fp4_swiglu, quantize_fp4
    g = gen(rows + n)
    experts = len(split) - 1
    x = torch.randn(rows, k, device="cuda", generator=g).to(torch.bfloat16)
    a = quantize_fp4(x, offsets=torch.tensor(split, device="cuda", dtype=torch.int32))
    w, up = weights(g, experts, n, k), weights(g, experts, n, k)
    out = torch.full((rows, n), 3.0, device="cuda", dtype=torch.bfloat16)
    assert (gemm_fp4_swiglu(a, w, up, out) if gated else gemm_fp4(a, w, out)) is out
    values, matrices, ups = nearest(x), held(w), held(up)
    for e, (lo, hi) in enumerate(zip(split, split[1:])):
        if lo == hi:
            continue
        if gated:
            want, tol = swiglu_reference(values[lo:hi], matrices[e], ups[e])
            assert bool(((out[lo:hi].double() - want).abs() <= tol).all())
        else:
            check_gemm(out[lo:hi], values[lo:hi], matrices[e])
    assert (out[:split[0]] == 3).all() and (out[split[-1]:] == 3).all()


def test_results_at_a_pitch_and_off_the_boundary():
    from hcomm_b200.ops.fp4 import gemm_fp4, quantize_fp4
    g = gen(21)
    a, b = quantize_fp4(spread(g, 150, 256)), weights(g, 200, 256)
    want = gemm_fp4(a, b)
    for pitch, first in ((208, 0), (208, 8), (203, 0), (208, 3)):
        big = torch.full((150, pitch), 9.0, device="cuda", dtype=torch.bfloat16)
        out = big.view(-1)[first:first + 149 * pitch + 200].as_strided((150, 200), (pitch, 1))
        gemm_fp4(a, b, out)
        assert torch.equal(out, want)
        keep = torch.ones_like(big, dtype=torch.bool)
        keep.view(-1)[first:].as_strided((150, 200), (pitch, 1))[:] = False
        assert (big[keep] == 9).all()


def test_a_block_that_is_no_number_reaches_its_row_only():
    from hcomm_b200.ops.fp4 import gemm_fp4, quantize_fp4
    g = gen(31)
    x = torch.randn(140, 256, device="cuda", generator=g)
    b = weights(g, 130, 256)
    clean = gemm_fp4(quantize_fp4(x), b)
    x[137, 77] = float("inf")
    out = gemm_fp4(quantize_fp4(x), b)
    assert torch.isnan(out[137]).all()
    out[137] = clean[137]
    assert torch.equal(out, clean)


def test_on_another_stream_and_in_a_replayed_graph():
    from hcomm_b200.ops.fp4 import gemm_fp4, quantize_fp4
    g = gen(41)
    x, b = spread(g, 200, 512), weights(g, 384, 512)
    first = gemm_fp4(quantize_fp4(x), b)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = gemm_fp4(quantize_fp4(x), b)
    stream.synchronize()
    assert torch.equal(first, other)
    offsets = torch.tensor([0, 100, 150], device="cuda", dtype=torch.int32)
    experts = weights(g, 2, 384, 512)
    out = torch.zeros(200, 384, device="cuda", dtype=torch.bfloat16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = gemm_fp4(quantize_fp4(x), b)
        gemm_fp4(quantize_fp4(x, offsets=offsets), experts, out)
    x.copy_(spread(g, 200, 512))
    offsets.copy_(torch.tensor([0, 7, 200], device="cuda", dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, gemm_fp4(quantize_fp4(x), b))
    for e, (lo, hi) in enumerate(((0, 7), (7, 200))):
        check_gemm(out[lo:hi], nearest(x[lo:hi]), held(experts)[e])


@pytest.mark.parametrize("m,n,k", [(1, 4096, 14336), (100, 1000, 4096), (16, 8192, 8192), (33, 130, 2080), (128, 1027, 5120), (200, 512, 8192)])
@pytest.mark.parametrize("gated", [False, True])
def test_tiles_that_ctas_share_along_k(m, n, k, gated):
    from hcomm_b200.ops.fp4 import gemm_fp4, gemm_fp4_swiglu, quantize_fp4
    g = gen(m + n + k)
    a = quantize_fp4(torch.randn(m, k, device="cuda", generator=g).to(torch.bfloat16))
    b, up = (quantize_fp4(torch.randn(n, k, device="cuda", generator=g) * 0.02) for _ in range(2))
    outs = [gemm_fp4_swiglu(a, b, up) if gated else gemm_fp4(a, b) for _ in range(3)]
    assert all(torch.equal(o, outs[0]) for o in outs)
    if gated:
        want, tol = swiglu_reference(held(a), held(b), held(up))
        assert bool(((outs[0].double() - want).abs() <= tol).all())
    else:
        check_gemm(outs[0], held(a), held(b))
    # an odd pitch: values one by one
    big = torch.zeros(m, n + 3, device="cuda", dtype=torch.bfloat16)
    (gemm_fp4_swiglu(a, b, up, big[:, 1:n + 1]) if gated else gemm_fp4(a, b, big[:, 1:n + 1]))
    assert torch.equal(big[:, 1:n + 1], outs[0]) and not big[:, 0].any() and not big[:, n + 1:].any()


@pytest.mark.parametrize("rows,n,k,split", [(8, 1024, 4096, [0, 1, 1, 3, 8]), (40, 500, 2080, [0, 0, 40]), (6, 256, 8192, [2, 2, 2, 2]), (130, 130, 1024, [0, 129, 130, 130]), (3, 1000, 768, [0] + [1] * 40)])
@pytest.mark.parametrize("gated", [False, True])
def test_tiles_of_experts_that_ctas_share_along_k(rows, n, k, split, gated):
    test_products_by_expert(rows, n, k, split, gated)


def test_refusals():
    from hcomm_b200.ops.fp4 import Fp4Tensor, dequantize_fp4, gemm_fp4, gemm_fp4_swiglu, quantize_fp4
    torch.cuda.set_device(0)
    x = torch.zeros(8, 128, device="cuda")
    fp8, scales = x.to(torch.float8_e4m3fn), torch.ones(8, 1, device="cuda")
    offsets = torch.tensor([0, 4, 8], device="cuda", dtype=torch.int32)
    for error, args, kw in ((TypeError, (x.double(),), {}), (TypeError, (x.int(),), {}), (TypeError, (fp8,), {}), (TypeError, (x, scales), {}), (ValueError, (x[0],), {}),
                            (ValueError, (x[:, :48],), {}), (ValueError, (x.t(),), {}), (ValueError, (fp8[:, :96], scales), {}), (ValueError, (fp8, scales[:4]), {}),
                            (ValueError, (fp8, scales.double()), {}), (ValueError, (x.cpu(),), {}), (ValueError, (x,), dict(offsets=offsets.long())),
                            (ValueError, (x,), dict(offsets=offsets[:1])), (ValueError, (x,), dict(offsets=offsets.cpu())), (ValueError, (x[None],), dict(offsets=offsets)),
                            (ValueError, (x,), dict(offsets=torch.zeros(1026, device="cuda", dtype=torch.int32)))):
        with pytest.raises(error):
            quantize_fp4(*args, **kw)
    q, w = quantize_fp4(x), quantize_fp4(torch.zeros(2, 16, 128, device="cuda"))
    b, grouped = quantize_fp4(torch.zeros(16, 128, device="cuda")), quantize_fp4(x, offsets=offsets)
    with pytest.raises(TypeError):
        dequantize_fp4(q, torch.float8_e4m3fn)
    with pytest.raises(ValueError):
        dequantize_fp4(Fp4Tensor(q.values, q.scales[:0]))
    wrong = quantize_fp4(torch.zeros(16, 96, device="cuda"))
    out = torch.zeros(8, 16, device="cuda", dtype=torch.bfloat16)
    for args in ((q, w), (grouped, b), (q, wrong), (q, grouped), (quantize_fp4(x, offsets=offsets[:2]), w), (w, b), (q, b, out.float()), (q, b, out[:, :8]), (q, b, out.t()),
                 (q, b, out[:1].expand(8, 16)), (q, b, out.cpu()), (Fp4Tensor(q.values[:, ::2], q.scales), b), (q, Fp4Tensor(b.values, b.scales[:0]))):
        with pytest.raises(ValueError):
            gemm_fp4(*args)
    with pytest.raises(TypeError):
        gemm_fp4(x, b)
    with pytest.raises(ValueError):
        gemm_fp4_swiglu(q, b, quantize_fp4(torch.zeros(32, 128, device="cuda")))
    assert gemm_fp4(quantize_fp4(x[:0]), b).shape == (0, 16)
    none = quantize_fp4(x[:0], offsets=torch.zeros(3, device="cuda", dtype=torch.int32))
    assert gemm_fp4(none, w).shape == (0, 16) and dequantize_fp4(none).shape == (0, 128)
    with pytest.raises(ValueError):
        gemm_fp4(quantize_fp4(x[:, :0]), quantize_fp4(torch.zeros(16, 0, device="cuda")))


def test_rows_wider_than_a_grid():
    from hcomm_b200.ops.fp4 import dequantize_fp4, quantize_fp4
    x = torch.randn(2, 32 * 200001, device="cuda", generator=gen(52)).to(torch.bfloat16)
    back = dequantize_fp4(quantize_fp4(x))
    for at in range(0, x.shape[1], 320000):
        assert same(back[:, at:at + 320000], nearest(x[:, at:at + 320000]))


def test_a_checkpoint_that_is_not_aligned():
    from hcomm_b200.ops.fp4 import Fp4Tensor, gemm_fp4, quantize_fp4
    g = gen(51)
    codes = torch.randint(0, 256, (1 + 40 * 48,), device="cuda", generator=g, dtype=torch.uint8)[1:].view(40, 48)
    w = Fp4Tensor.from_parts(codes, torch.randint(120, 130, (40, 3), device="cuda", generator=g, dtype=torch.uint8))
    a = quantize_fp4(spread(g, 5, 96))
    check_gemm(gemm_fp4(a, w), held(a), held(w))


FIRST_CALLS = """
import sys
sys.path.insert(0, {root!r})
import torch
from hcomm_b200.ops.fp4 import gemm_fp4, quantize_fp4
from hcomm_b200.ops.router import route
x = torch.randn({m}, 512, device="cuda").to(torch.bfloat16)
w = torch.randn(2048, 512, device="cuda").to(torch.bfloat16)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = gemm_fp4(quantize_fp4(x), quantize_fp4(w))
    r = route(y[:, :64], 4)
graph.replay()
torch.cuda.synchronize()
assert torch.equal(y, gemm_fp4(quantize_fp4(x), quantize_fp4(w))) and torch.equal(r.topk_idx, route(y[:, :64], 4).topk_idx)
print("same")
"""


@pytest.mark.parametrize("m", [20, 6000])
def test_first_calls_of_a_process_are_captured(m):
    import subprocess
    import sys
    from pathlib import Path
    root = str(Path(__file__).resolve().parent.parent)
    res = subprocess.run([sys.executable, "-c", FIRST_CALLS.format(root=root, m=m)], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and "same" in res.stdout, res.stdout + res.stderr


def test_threads_and_streams_at_the_same_time():
    import threading
    from hcomm_b200.ops.fp4 import gemm_fp4, quantize_fp4, take_kernel_error
    g = gen(61)
    w = weights(g, 1024, 1024)
    xs = [torch.randn(m, 1024, device="cuda", generator=g).to(torch.bfloat16) for m in (1, 40, 300, 2000)]
    want = [gemm_fp4(quantize_fp4(x), w) for x in xs]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        torch.cuda.set_device(0)
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                if not torch.equal(gemm_fp4(quantize_fp4(xs[i]), w), want[i]):
                    bad.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(xs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad and take_kernel_error() == 0


def test_depths_beyond_32_bits_are_refused_by_every_way():
    import contextlib
    from hcomm_b200.ops.fp4 import Fp4Tensor, gemm_fp4, gemm_fp4_swiglu
    torch.cuda.set_device(0)
    k = 2 ** 31 - 128
    q = Fp4Tensor(torch.empty(1, k // 2, device="cuda", dtype=torch.uint8), torch.empty(k // 128, 512, device="cuda", dtype=torch.uint8))         # 10 GB
    for mode in (contextlib.nullcontext(), torch.overrides.BaseTorchFunctionMode()):        # the native call, and the general one
        with mode:
            with pytest.raises(ValueError, match="at most"):
                gemm_fp4(q, q)
            with pytest.raises(ValueError, match="at most"):
                gemm_fp4_swiglu(q, q, q)


def fp8_rows(g, rows, cols, scales):
    """Codes of every kind but NaN, and scales [rows, cols // 128] of the given kind."""
    codes = torch.randint(0, 256, (rows, cols), device="cuda", generator=g, dtype=torch.uint8)
    codes[(codes & 127) == 127] = 3
    return codes.view(torch.float8_e4m3fn), scales.expand(rows, cols // 128).float().contiguous()


@pytest.mark.parametrize("offsets", [None, [0, 3, 3, 140, 150]])
@pytest.mark.parametrize("low,high", [(-149, -120), (-127, -100), (-80, -55), (-66, -62), (100, 118)])
def test_exchanged_rows_of_every_magnitude(low, high, offsets):
    """Products below the range of ordinary numbers, and on both sides of the border (block scales of 2^-63) where the multiplier is taken into the
    block's power of two instead of into every value; scales that are no powers of two, and negative ones."""
    from hcomm_b200.ops.fp4 import dequantize_fp4, quantize_fp4
    g = gen(71 - low)
    rows, cols = 150, 512
    power = torch.randint(low, high + 1, (rows, cols // 128), device="cuda", generator=g)
    mantissa = 1 + torch.rand(rows, cols // 128, device="cuda", generator=g, dtype=torch.float64)
    sign = torch.where(torch.rand(rows, cols // 128, device="cuda", generator=g) < 0.3, -1.0, 1.0)
    x, scales = fp8_rows(g, rows, cols, (sign * torch.ldexp(mantissa, power)).float())
    # blocks of small codes beside the others, so that the largest product is far below 448 of its scale
    small = torch.randint(0, 9, (rows, cols), device="cuda", generator=g, dtype=torch.uint8) + 128 * torch.randint(0, 2, (rows, cols), device="cuda", generator=g, dtype=torch.uint8)
    pick = (torch.rand(rows, cols // 32, device="cuda", generator=g) < 0.4).repeat_interleave(32, 1)
    x = torch.where(pick, small, x.view(torch.uint8)).view(torch.float8_e4m3fn)
    want = nearest((x.double() * scales.double().repeat_interleave(128, 1)).float())        # a value is the product rounded to fp32, once
    at = None if offsets is None else torch.tensor(offsets, device="cuda", dtype=torch.int32)
    q = quantize_fp4(x, scales, offsets=at)
    assert same(dequantize_fp4(q, torch.float32), want)
    if at is None:
        assert same(held(q), want)
        border = q.block_scales()
        assert (low, high) != (-80, -55) or ((border == 63).any() and (border == 64).any())


@pytest.mark.parametrize("offsets", [None, [0, 3, 3, 140, 150]])
def test_exchanged_rows_that_are_no_numbers(offsets):
    from hcomm_b200.ops.fp4 import dequantize_fp4, quantize_fp4
    g = gen(72)
    x, scales = fp8_rows(g, 150, 512, torch.ones(150, 4, device="cuda"))
    for row, value in enumerate((0.0, -0.0, float("inf"), float("-inf"), float("nan"), torch.finfo(torch.float32).max, -torch.finfo(torch.float32).max, 1e-45, 2.0 ** -126)):
        scales[10 + row, 1], scales[60 + row, :] = value, value
    x.view(torch.uint8)[100, 40], x.view(torch.uint8)[101, 511], x.view(torch.uint8)[102, :32] = 0x7f, 0xff, 0x7f
    x.view(torch.uint8)[62, 128:256] = 0          # no numbers: zero times infinity
    scales[103, 0], x.view(torch.uint8)[103, 5] = 0.0, 0x7f
    want = nearest((x.double() * scales.double().repeat_interleave(128, 1)).float())
    at = None if offsets is None else torch.tensor(offsets, device="cuda", dtype=torch.int32)
    q = quantize_fp4(x, scales, offsets=at)
    assert same(dequantize_fp4(q, torch.float32), want)
    bad = torch.isnan(want.view(150, 16, 32)).any(2)
    for row, blocks in ((12, 4), (13, 4), (14, 4), (62, 16), (63, 16), (64, 16), (100, 1), (101, 1), (102, 1), (103, 1), (10, 0), (11, 0), (60, 0), (67, 0)):
        assert int(bad[row].sum()) == blocks, row


@pytest.mark.parametrize("m,n,k,grouped", [(9, 40, 64, False), (1, 256, 8192, False), (300, 136, 96, False), (1000, 1000, 64, True)])
def test_gates_far_below_zero(m, n, k, grouped):
    """silu is 0 below -87.3, where its magnitude is under 2^-119: beside what a gated product is off by anyway, up times that.  Infinite gates give what
    the formula gives."""
    from hcomm_b200.ops.fp4 import Fp4Tensor, gemm_fp4_swiglu, quantize_fp4
    g = gen(m + n)
    x = torch.randn(m, k, device="cuda", generator=g)
    gate, up = torch.randn(n, k, device="cuda", generator=g), torch.randn(n, k, device="cuda", generator=g)
    spread_out = torch.tensor([-60.0, -80.0, -86.0, -88.0, -90.0, -200.0, -3e4, 90.0, 3e4], device="cuda")
    x[:, :32] = 0
    x[:, 0] = 4.0
    gate[:, :32] = 0
    gate[:, 0] = spread_out[torch.arange(n, device="cuda") % 9] / 4.0
    gate[:, 32:] *= 2.0 ** -6
    a, w, u = quantize_fp4(x), quantize_fp4(gate), quantize_fp4(up)
    args = (a, w, u)
    if grouped:
        args = (quantize_fp4(x, offsets=torch.tensor([0, m], device="cuda", dtype=torch.int32)), *(Fp4Tensor(q.values[None], q.scales) for q in (w, u)))
    out = gemm_fp4_swiglu(*args).double()
    want, tol = swiglu_reference(held(a), held(w), held(u))
    ups = (held(a) @ held(u).t()).abs() + k * 2.0 ** -23 * (held(a).abs() @ held(u).abs().t())
    far = (held(a) @ held(w).t()) < -80
    assert far.any() and bool(((out - want).abs() <= tol + far * 2.0 ** -119 * ups).all())
    # beyond the range of 32 bits
    huge = torch.zeros(2, k, device="cuda")
    huge[:, 0] = torch.tensor([3e38, -3e38], device="cuda")
    x[:] = 0
    x[:, 0], x[:, 1] = 2.0 ** 10, 1.0
    up[:] = 0
    up[:, 1] = 3.0
    # the one shares its power of two, 2^8, with the 2^10 and becomes 0: infinity times up's 0, and -inf 0
    assert torch.isnan(gemm_fp4_swiglu(quantize_fp4(x), quantize_fp4(huge), quantize_fp4(up[:2]))).all()
    x[:, 40], up[:, 40] = 1.0, 3.0          # a block of their own: up is 3
    out = gemm_fp4_swiglu(quantize_fp4(x), quantize_fp4(huge), quantize_fp4(up[:2]))
    assert (out[:, 0] == float("inf")).all() and torch.isnan(out[:, 1]).all()          # inf 1 3; -inf 0


def test_the_deepest_product():
    """As deep as a product may be: a row of 2^31 - 288 columns by itself, nothing but its first and last blocks filled."""
    from hcomm_b200.ops.fp4 import Fp4Tensor, gemm_fp4, gemm_fp4_swiglu, take_kernel_error
    torch.cuda.set_device(0)
    k = 2 ** 31 - 288
    values = torch.zeros(1, k // 2, device="cuda", dtype=torch.uint8)
    values[0, :16], values[0, -16:] = 0x22, 0x44            # 32 ones, 32 twos
    q = Fp4Tensor(values, torch.full((-(-k // 128), 512), 127, device="cuda", dtype=torch.uint8))         # 10 GB
    assert gemm_fp4(q, q).item() == 32 + 4 * 32
    assert gemm_fp4_swiglu(q, q, q).item() == 160 * 160
    assert take_kernel_error() == 0
    del q, values
    torch.cuda.empty_cache()
