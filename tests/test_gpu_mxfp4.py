"""MXFP4 kernels against the format's definition in 64 bits: quantizers bit for bit, products within the roundings they make."""
import pytest
import torch

from eider_b200 import ops
from tests import mxfp4_reference as ref
from tests.util import require_cuda

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _cuda():
    require_cuda()


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def check_matrix(m, x):
    """Codes and scales of a quantized matrix against the definition, padding included."""
    codes, scales = ref.quantize(x)
    got, clean = ref.untile(m.scales, m.rows, m.k)
    assert torch.equal(got, scales)
    assert clean, "padding scales are not zero"
    finite = (scales != 255).repeat_interleave(32, 1)  # (the codes of a NaN block mean nothing)
    assert torch.equal(ref.unpack(m.packed)[finite], codes[finite])


# ---- quantisation -----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,k", [(1, 32), (1, 5120), (3, 96), (31, 128), (130, 160), (257, 2880), (512, 64), (1029, 416)])
def test_quantize_is_exact(rows, k, dtype):
    x = randn(gen(rows + k), rows, k, dtype=dtype, std=3.0)
    m = ops.quantize_mxfp4(x)
    check_matrix(m, x)
    codes, scales = ref.quantize(x)
    for out in (torch.float32, torch.bfloat16):
        assert torch.equal(m.dequantize(out).double(), ref.values(codes, scales))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantize_boundaries(dtype):
    """Ties between codes, saturation between 6 and 8, zeros of both signs, magnitudes from subnormal to the largest."""
    steps = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 6.5, 7.0, 7.75, 0.0, -0.0, 0.125, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, -7.5,
                          0.2490234375, 0.251953125, 4.96875, 5.03125, 1.0, 2.0, 3.0, 4.0, 0.5, -6.0], device="cuda")
    exponents = [-148, -140, -133, -130, -128, -127, -126, -125, -120, -60, -2, 0, 1, 60, 120, 124, 125]
    x = torch.stack([(steps.double() * 2.0 ** e).to(dtype) for e in exponents])
    x = torch.cat([x, torch.zeros_like(x[:1]), -torch.zeros_like(x[:1])])
    x = x[torch.isfinite(x).all(1)]
    check_matrix(ops.quantize_mxfp4(x.contiguous()), x)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantize_poisoned_blocks(dtype):
    x = randn(gen(3), 70, 160, dtype=dtype)
    x[1, 33] = float("nan")
    x[2, 0] = float("inf")
    x[69, 159] = -float("inf")
    m = ops.quantize_mxfp4(x)
    check_matrix(m, x)
    bad = torch.isnan(m.dequantize())
    assert bad[1, 32:64].all() and bad[2, :32].all() and bad[69, 128:].all() and int(bad.sum()) == 96


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantize_strides_and_alignment(dtype):
    wide = randn(gen(4), 40, 500, dtype=dtype)
    for x in (wide[:, :96], wide[:, 3:131], wide[::2, 8:40], wide.flatten()[1:1 + 3 * 64].reshape(3, 64)):
        check_matrix(ops.quantize_mxfp4(x), x)
    one = wide[5:6, 7:39]  # one row: its stride does not matter
    check_matrix(ops.quantize_mxfp4(one), one)


def test_weight_quantizer_and_layouts():
    g = gen(5)
    for n, k in ((1, 32), (130, 96), (200, 2912)):
        w = randn(g, n, k, std=0.02)
        m = ops.Mxfp4Weight.quantize(w)
        codes, scales = ref.quantize(w)
        assert torch.equal(ref.unpack(m.packed), codes) and torch.equal(m.scales_row_major, scales)
        tiled, clean = ref.untile(m.scales_tiled, n, k)
        assert torch.equal(tiled, scales) and clean
        assert torch.equal(m.scales_rows[:, : k // 32], scales) and not m.scales_rows[:, k // 32:].any() and m.scales_rows.shape[1] % 16 == 0
        assert torch.equal(m.dequantize().double(), ref.values(codes, scales))


def test_silu_quantizer():
    """The fused producer's values are those of SiLU * up but for codes next to a boundary (f32 exponential and reciprocal)."""
    for rows, k in ((1, 32), (5, 96), (130, 2784)):
        x = randn(gen(k), rows, 2 * k, std=2.0)
        m = ops.silu_mul_halves_quantize_mxfp4(x)
        act = ref.silu_mul(x.double())
        codes, scales = ref.quantize(act)
        got, clean = ref.untile(m.scales, rows, k)
        assert clean
        # a boundary is met by about 1e-5 of the values at a relative error of 1e-6; none may be off by more than a step
        assert (got != scales).float().mean() <= 1e-3 and (ref.unpack(m.packed) != codes).float().mean() <= 1e-3
        step = torch.exp2(scales.double() - 127).repeat_interleave(32, 1) * 2
        assert ((m.dequantize().double() - act).abs() <= step * 1.01).all()


# ---- dense product ------------------------------------------------------------------------------------------------
def product_bound(x, w, extra=0):
    """f32 sums of exact products: the tensor core adds 64 products at a time to what it has, each addition off by at most a step of
    the sum (2^-23 of the largest partial sum, which sum |x w| bounds)."""
    return (x.shape[1] // 64 + 4 + extra) * 2.0 ** -23 * (x.abs() @ w.abs().t())


def rounded(bound, y, dtype):
    """... and the result rounded to its type."""
    return bound + torch.finfo(dtype).eps / 2 * y.abs()


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,k,n", [(1, 32, 1), (1, 5120, 320), (5, 96, 40), (64, 160, 136), (129, 224, 264), (300, 2912, 1000), (520, 512, 1296)])
def test_gemm(m, k, n, out):
    g = gen(m + k + n)
    x = randn(g, m, k)
    xq, w = ops.quantize_mxfp4(x), ops.Mxfp4Weight.from_checkpoint(*ref.weight(g, n, k))
    xv, wv = ref.values(*ref.quantize(x)), w.dequantize().double()
    plan = ops.Mxfp4MatmulPlan(m, n, k)
    y = plan.run(xq, w, alpha=0.75, out_dtype=out)
    want = 0.75 * (xv @ wv.t())
    assert ((y.double() - want).abs() <= rounded(product_bound(xv, wv), want, out)).all()
    c = randn(g, m, n, dtype=out)
    y = plan.run(xq, w, beta=-0.5, c=c, out_dtype=out)
    want = xv @ wv.t() - 0.5 * c.double()
    assert ((y.double() - want).abs() <= rounded(product_bound(xv, wv, 2) + 2.0 ** -23 * c.double().abs(), want, out)).all()
    assert plan.status() == 0


@pytest.mark.parametrize("block_n", [64, 128, 192, 256, 384, 512])
def test_gemm_tiles_agree(block_n):
    """Every tile shape adds the same products in the same order."""
    g = gen(7)
    for m, k, n in ((300, 1184, 840), (128, 256, 512)):
        xq, w = ops.quantize_mxfp4(randn(g, m, k)), ops.Mxfp4Weight.from_checkpoint(*ref.weight(g, n, k))
        plan = ops.Mxfp4MatmulPlan(m, n, k)
        plan.set_block_n(64)
        want = plan.run(xq, w, out_dtype=torch.float32)
        plan.set_block_n(block_n)
        assert torch.equal(plan.run(xq, w, out_dtype=torch.float32), want)
        assert torch.equal(plan.run(xq, w), want.to(torch.bfloat16))
        assert plan.status() == 0


def test_gemm_scale_range():
    """Every scale from 2^-126 to 2^126 that a product can hold, and NaN scales in one row of each operand."""
    g = gen(8)
    m, k, n = 40, 128, 72
    codes = torch.randint(0, 16, (m, k), generator=g, device="cuda", dtype=torch.uint8)
    sx = torch.randint(1, 254, (m, 1), generator=g, device="cuda").expand(m, k // 32).contiguous().to(torch.uint8)
    wp, _ = ref.weight(g, n, k)
    sw = torch.full((n, k // 32), 127, dtype=torch.uint8, device="cuda")
    sw[1] = 255
    sx[2, 3] = 255
    x = ops.Mxfp4Matrix(ref.pack(codes).contiguous(), ops._mxfp4_tiled(sx, 1, m, k), m, k)
    w = ops.Mxfp4Weight.from_checkpoint(wp, sw)
    y = ops.Mxfp4MatmulPlan(m, n, k).run(x, w, out_dtype=torch.float32)
    xv, wv = ref.values(codes, sx), ref.values(ref.unpack(wp), sw)
    want = xv @ wv.t()
    assert torch.isnan(y[2]).all() and torch.isnan(y[:, 1]).all()
    fine = ~torch.isnan(want) & (want.abs() < 3e38)
    assert ((y.double() - want).abs()[fine] <= (product_bound(xv, wv) + 2.0 ** -126)[fine]).all()


@pytest.mark.parametrize("rows", [1, 127, 130, 513])
def test_gated_gemm_equals_two_launches(rows):
    g = gen(rows)
    for inter, k in ((128, 96), (384, 2048)):
        xq, w = ops.quantize_mxfp4(randn(g, rows, k)), ops.Mxfp4Weight.from_checkpoint(*ref.weight(g, 2 * inter, k, std=0.1))
        plan = ops.Mxfp4MatmulPlan(rows, 2 * inter, k)
        fused = plan.run_silu_quantize(xq, w)
        staged = ops.silu_mul_halves_quantize_mxfp4(plan.run(xq, w, out_dtype=torch.float32))
        assert torch.equal(fused.packed, staged.packed) and torch.equal(fused.scales, staged.scales)
        assert plan.status() == 0


@pytest.mark.parametrize("rows,hidden,inter", [(1, 96, 160), (77, 512, 288), (300, 512, 384)])
def test_ffn(rows, hidden, inter):
    """DenseFfn over MXFP4 weights: the activation's codes against 64 bits but for boundaries, then its product exactly."""
    g = gen(rows)
    gate_up, down = (ops.Mxfp4Weight.from_checkpoint(*ref.weight(g, n, k, std=0.1)) for n, k in ((2 * inter, hidden), (hidden, inter)))
    x, residual = randn(g, rows, hidden, dtype=torch.bfloat16), randn(g, rows, hidden, dtype=torch.bfloat16)
    y = ops.DenseFfn(gate_up, down).run(x, residual)
    act = ref.silu_mul(ref.values(*ref.quantize(x)) @ gate_up.dequantize().double().t())
    act = ref.values(*ref.quantize(act))
    wv = down.dequantize().double()
    want = act @ wv.t() + residual.double()
    # one code in a thousand may be a step (a third of its value) off: sqrt(1e-3) / 3 of the product's size, and the rounding
    off = (y.double() - want).abs()
    assert (off <= 0.05 * (act.abs() @ wv.abs().t()) + 2.0 ** -8 * want.abs()).all()
    assert off.norm() <= (0.011 + 2.0 ** -8) * want.norm()


# ---- few tokens -----------------------------------------------------------------------------------------------
def decode_bound(x, w, dtype):
    """Block sums of two (f32: four) MMAs, K / 32 of them added up in f32 and eleven warps' sums after them; f32 activations go in as
    two f16 terms that leave 2^-23 of an element; elements far below their token's largest leave 2^-32 of that."""
    total = x.abs() @ w.abs().t()
    steps = x.shape[1] // 32 + 16 + (1 if dtype == torch.float32 else 0)
    return steps * 2.0 ** -23 * total + 2.0 ** -32 * x.abs().amax(1, keepdim=True) * w.abs().sum(1)


SHAPES = [(1, 32), (40, 96), (256, 512), (1000, 2912), (6150, 1056), (3001, 8192), (15000, 288)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens", [1, 2, 3, 4, 5, 8, 9, 16, 17, 31, 33, 64])
def test_decode(tokens, dtype):
    g = gen(tokens)
    for n, k in SHAPES:
        x, w = randn(g, tokens, k, dtype=dtype), ops.Mxfp4Weight.from_checkpoint(*ref.weight(g, n, k))
        wv, xv = w.dequantize().double(), x.double()
        want, bound = xv @ wv.t(), decode_bound(xv, wv, dtype)
        plan = ops.Mxfp4DecodePlan(64, n, k)
        for out in (torch.float32, torch.bfloat16):
            y = plan.run(x, w, out_dtype=out)
            assert y.shape == (tokens, n)
            assert ((y.double() - want).abs() <= rounded(bound, want, out)).all(), (n, k, out)
        c = randn(g, tokens, n)
        y = plan.run(x, w, beta=0.25, c=c, out_dtype=torch.float32)
        assert ((y.double() - want - 0.25 * c.double()).abs() <= bound + 2.0 ** -22 * (want.abs() + c.double().abs())).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_decode_activation_ranges(dtype):
    """Tokens whose elements start at zero, grow or shrink by many powers of two along K, or are tiny or huge throughout."""
    g = gen(11)
    n, k = 200, 5120
    x = torch.randn(14, k, generator=g, device="cuda")
    ramp = torch.linspace(0, 1, k, device="cuda")
    x[0, :3000] = 0
    x[1, 300:] = 0
    x[2] = 0
    x[3] *= torch.exp2(60 * ramp)
    x[4] *= torch.exp2(-60 * ramp)
    x[5] *= 2.0 ** -120
    x[6] *= 2.0 ** 100
    x[7, ::2] = 0
    x[8, :5000] *= 2.0 ** -100
    x[9, 40] = 2.0 ** 90
    x[10] *= torch.exp2(torch.randint(-40, 40, (k,), generator=g, device="cuda").float())
    x[11, :] = 0
    x[11, -1] = 1.0
    x[12] = 2.0 ** -126
    x = x.to(dtype)
    w = ops.Mxfp4Weight.from_checkpoint(*ref.weight(g, n, k))
    wv, xv = w.dequantize().double(), x.double()
    y = ops.Mxfp4DecodePlan(16, n, k).run(x, w, out_dtype=torch.float32).double()
    assert ((y - xv @ wv.t()).abs() <= decode_bound(xv, wv, dtype) + 2.0 ** -140).all()
    assert not y[2].any()


@pytest.mark.parametrize("k,dtype", [(1024, torch.bfloat16), (1024, torch.float32), (1056, torch.bfloat16), (1056, torch.float32)])
def test_decode_poison_stays_with_its_token_and_row(k, dtype):
    g = gen(12)
    n = 100
    wp, ws = ref.weight(g, n, k)
    ws[7, 3] = 255
    ws[9] = 0
    ws[11, 5] = 254
    w = ops.Mxfp4Weight.from_checkpoint(wp, ws)
    x = randn(g, 5, k, dtype=dtype)
    x[1, 100] = float("nan")
    x[3, 700] = float("inf")
    y = ops.Mxfp4DecodePlan(8, n, k).run(x, w, out_dtype=torch.float32)
    wv = ref.values(ref.unpack(wp), ws)
    want = x.double() @ wv.t()
    assert torch.isnan(y[1]).all() and not torch.isfinite(y[3]).any() and torch.isnan(y[:, 7]).all()
    fine = torch.isfinite(want) & (want.abs() < 3e38)
    fine[:, 7] = False
    assert fine[0].sum() >= 98 and ((y.double() - want).abs()[fine] <= (decode_bound(x.double().nan_to_num(0, 0, 0), wv.nan_to_num(0), dtype) + 1e-38)[fine]).all()
    # infinities by the weight's sign, NaN where it is zero (row 11 aside: what its scale of 2^127 makes of the finite elements overflows)
    rest = torch.arange(n, device="cuda") != 11
    assert torch.equal(y[3, rest].double().nan_to_num(nan=7.0), want[3, rest].nan_to_num(nan=7.0))


@pytest.mark.parametrize("tokens,dtype", [(1, torch.bfloat16), (2, torch.float32), (4, torch.bfloat16), (8, torch.float32), (16, torch.bfloat16), (40, torch.bfloat16)])
def test_decode_is_the_same_in_every_run_and_order(tokens, dtype):
    """Two runs agree bit for bit, and a token's result depends neither on its place nor on the tokens beside it."""
    g = gen(13)
    n, k = 6150, 4064
    x, w = randn(g, tokens, k, dtype=dtype), ops.Mxfp4Weight.from_checkpoint(*ref.weight(g, n, k))
    plan = ops.Mxfp4DecodePlan(64, n, k)
    y = plan.run(x, w, out_dtype=torch.float32)
    assert torch.equal(plan.run(x, w, out_dtype=torch.float32), y)
    order = torch.randperm(tokens, generator=g, device="cuda")
    assert torch.equal(plan.run(x[order], w, out_dtype=torch.float32), y[order])
    x[1:] *= 2.0 ** 30
    assert torch.equal(plan.run(x, w, out_dtype=torch.float32)[0], y[0])


def test_calls_in_a_row_read_what_was_just_written():
    """Calls without a pause between them, on buffers that the allocator hands around and that held NaNs before: every launch reads what the
    one in front of it wrote, not what was there when it started."""
    g = gen(14)
    for n, k, tokens, dtype in ((3001, 8192, 9, torch.float32), (1000, 2912, 8, torch.bfloat16), (256, 512, 3, torch.float32)):
        w, plan = ops.Mxfp4Weight.from_checkpoint(*ref.weight(g, n, k)), ops.Mxfp4DecodePlan(64, n, k)
        gemm = ops.Mxfp4MatmulPlan(tokens, n, k)
        xs = [randn(g, tokens, k, dtype=dtype) for _ in range(2)]
        want = []
        for x in xs:
            want.append((plan.run(x, w), gemm.run(ops.quantize_mxfp4(x), w), ops.quantize_mxfp4(x).dequantize()))
            torch.cuda.synchronize()
        wrong = torch.zeros((), device="cuda", dtype=torch.int64)
        for i in range(100):
            junk = torch.full((tokens * k // 2,), float("nan"), device="cuda", dtype=torch.float64)
            junk.sum()
            del junk
            x, (decoded, multiplied, values) = xs[i % 2], want[i % 2]
            wrong += (plan.run(x, w) != decoded).any().long()
            wrong += (gemm.run(ops.quantize_mxfp4(x), w) != multiplied).any().long()
            wrong += (ops.quantize_mxfp4(x).dequantize() != values).any().long()
        assert int(wrong) == 0


# ---- routed experts -----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens,experts,top_k,hidden,inter", [(1, 4, 2, 64, 32), (5, 8, 3, 160, 96), (77, 16, 4, 512, 288), (300, 6, 6, 288, 320), (1000, 32, 2, 256, 128)])
def test_experts(tokens, experts, top_k, hidden, inter, dtype):
    g = gen(tokens)
    gate_up, down = ([t.reshape(experts, -1, t.shape[1]) for t in ref.weight(g, experts * n, k, std=0.1)] for n, k in ((2 * inter, hidden), (hidden, inter)))
    gu, dn = ops.GroupedMxfp4Weights.from_checkpoint(*gate_up), ops.GroupedMxfp4Weights.from_checkpoint(*down)
    x, logits = randn(g, tokens, hidden, dtype=dtype), randn(g, tokens, experts)
    logits[:, 1] -= 20  # an expert that (almost) nobody picks
    moe = ops.GroupedMoe(tokens, experts, top_k, hidden, inter, weight_format="mxfp4")
    y = moe.run(x, logits, gu, dn, w_gate_up_interleaved=gu.interleave_gate_up())
    y16 = moe.run(x, logits, gu, dn, w_gate_up_interleaved=gu.interleave_gate_up(), out_dtype=torch.bfloat16)
    assert torch.equal(y16, y.to(torch.bfloat16))
    xv = ref.values(*ref.quantize(x))
    gv, dv = ref.values(ref.unpack(gate_up[0]), gate_up[1]), ref.values(ref.unpack(down[0]), down[1])
    # the routes' rows as the layer left them: quantized inputs exactly, activations but for boundaries
    order, expert = moe.routes.sorted_routes.long(), moe.routes.sorted_experts.long()
    first = moe.routes.expert_offsets.long()
    for name, rows_of in (("gate_up_in", hidden), ("down_in", inter)):
        buffer = getattr(moe, name)
        blocks, group = rows_of // 32, (rows_of // 32 + 3) // 4
        tiles = buffer.scales.reshape(-1, group, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-1, group * 4)  # [tile * 128 + row][block]
        at = ((first[expert] + 127) // 128 + expert) * 128 + torch.arange(len(order), device="cuda") - first[expert]
        got = ref.values(ref.unpack(buffer.packed), tiles[at][:, :blocks])
        if name == "gate_up_in":
            assert torch.equal(got, xv[order // top_k])
        else:
            act = ref.silu_mul(torch.stack([xv[r // top_k] @ gv[e].t() for r, e in zip(order.tolist(), expert.tolist())]))
            codes, scales = ref.quantize(act)
            assert (got != ref.values(codes, scales)).double().mean() <= 2e-3
            step = torch.exp2(scales.double() - 127).repeat_interleave(32, 1) * 2
            assert ((got - act).abs() <= step * 1.01).all()
            act = got
    rows = torch.stack([act[i] @ dv[e].t() for i, e in enumerate(expert.tolist())])
    bound = torch.stack([act[i].abs() @ dv[e].abs().t() for i, e in enumerate(expert.tolist())]) * (inter // 64 + 4) * 2.0 ** -23 + 2.0 ** -8 * rows.abs()
    assert ((moe.down_out.double() - rows).abs() <= bound).all()
    weights = torch.softmax(logits.double().topk(top_k, 1)[0], 1).reshape(-1, 1)
    back, slack = torch.empty_like(rows), torch.empty_like(rows)
    back[order], slack[order] = rows, bound
    want = (back * weights).reshape(tokens, top_k, -1).sum(1)
    limit = ((slack + 2.0 ** -20 * back.abs()) * weights).reshape(tokens, top_k, -1).sum(1)
    assert ((y.double() - want).abs() <= limit + 1e-30).all()
    assert moe.gate_up_plan.status() == 0 and moe.down_plan.status() == 0


# ---- as they are used ---------------------------------------------------------------------------------------------
def test_streams_and_graphs():
    """Calls on a stream of their own, captured and replayed on new inputs; two graphs of one decode plan in flight together."""
    g = gen(21)
    n, k = 1000, 2048
    w = [ops.Mxfp4Weight.from_checkpoint(*ref.weight(g, n, k)) for _ in range(2)]
    plan, gemm = ops.Mxfp4DecodePlan(8, n, k), ops.Mxfp4MatmulPlan(8, n, k)
    x = [randn(g, 8, k, dtype=torch.bfloat16) for _ in range(2)]
    want = [(plan.run(x[i], w[i]), gemm.run(ops.quantize_mxfp4(x[i]), w[i])) for i in range(2)]
    torch.cuda.synchronize()
    streams, graphs, held, outs = [torch.cuda.Stream() for _ in range(2)], [], [torch.zeros_like(x[0]) for _ in range(2)], []
    for i, s in enumerate(streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            outs.append((plan.run(held[i], w[i]), gemm.run(ops.quantize_mxfp4(held[i]), w[i])))
        graphs.append(graph)
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                held[i].copy_(x[i])
                graphs[i].replay()
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(outs[i][0], want[i][0]) and torch.equal(outs[i][1], want[i][1])


def test_refusals():
    g = gen(22)
    w = ops.Mxfp4Weight.from_checkpoint(*ref.weight(g, 64, 96))
    x = randn(g, 4, 96)
    for bad in (x.half(), x.t(), x[:, :80], x[:0], x[0]):
        with pytest.raises(ops.ShapeError):
            ops.quantize_mxfp4(bad)
    with pytest.raises(ops.ShapeError):
        ops.quantize_mxfp4(x[:1].expand(4, 96))
    plan, gemm = ops.Mxfp4DecodePlan(4, 64, 96), ops.Mxfp4MatmulPlan(4, 64, 96)
    for args in ({"x": x[:, :64]}, {"x": randn(g, 5, 96)}, {"x": x.half()}, {"x": x.cpu()}, {"x": x, "out": torch.empty(4, 63, device="cuda")},
                 {"x": x, "beta": 1.0, "c": torch.empty(4, 64, device="cuda").half()}, {"x": x, "out_dtype": torch.float16}, {"x": x[:0]}):
        with pytest.raises(ops.ShapeError):
            plan.run(w=w, **args)
    xq = ops.quantize_mxfp4(x)
    with pytest.raises(ops.ShapeError):
        gemm.run(ops.quantize_mxfp4(x[:2]), w)
    with pytest.raises(ops.ShapeError):
        gemm.run(xq, w, out=torch.empty(4, 64, device="cuda", dtype=torch.float16))
    with pytest.raises(ops.ShapeError):
        gemm.run_silu_quantize(xq, w)
    with pytest.raises(ops.ShapeError):
        ops.Mxfp4DecodePlan(65, 64, 96)
    moe = ops.GroupedMoe(4, 2, 1, 64, 32, weight_format="mxfp4")
    with pytest.raises(ops.ShapeError):
        moe.run(randn(g, 4, 64), randn(g, 4, 2), None, None)


def test_combine_refuses_a_bf16_output_of_another_shape():
    rows = torch.zeros(8, 64, device="cuda", dtype=torch.bfloat16)
    weights = torch.zeros(4, 2, device="cuda")
    with pytest.raises(ops.ShapeError):
        ops.moe_weighted_accumulate(None, weights, rows, 4, 2, out=torch.zeros(3, 64, device="cuda", dtype=torch.bfloat16))


def test_decode_plans_report_their_status():
    """Poisoned activations give NaN with a status of 0: only a wait that ran out sets it."""
    g = gen(23)
    for tokens, k in ((1, 96), (9, 512)):  # one of each form
        plan, w = ops.Mxfp4DecodePlan(16, 200, k), ops.Mxfp4Weight.from_checkpoint(*ref.weight(g, 200, k))
        assert plan.status() == 0
        x = randn(g, tokens, k)
        x[0, 3] = float("nan")
        assert torch.isnan(plan.run(x, w)[0]).all() and plan.status() == 0


def block_bound(x, w, dtype):
    """decode_bound without its allowance for the token's largest element: what an element loses is at most 2^-22 (bf16, beyond 2^14 below) or
    2^-37 (f32) of the largest of its own block of 32."""
    steps = x.shape[1] // 32 + 16 + (1 if dtype == torch.float32 else 0)
    largest = x.abs().reshape(x.shape[0], -1, 32).amax(-1)
    lost = 2.0 ** -22 if dtype == torch.bfloat16 else 2.0 ** -37
    return steps * 2.0 ** -23 * (x.abs() @ w.abs().t()) + lost * largest @ w.abs().reshape(w.shape[0], -1, 32).sum(-1).t()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens,k", [(1, 1024), (2, 1024), (3, 96), (4, 1024), (5, 1056), (9, 2912), (16, 544), (33, 1056), (9, 1024), (24, 2048), (64, 1024)])
def test_decode_keeps_blocks_far_below_an_outlier(tokens, k, dtype):
    """An activation with one huge element that the weights do not look at (zero codes in its block): what is left of the results are blocks
    2^41 to 2^100 below it, in either form of the product."""
    g = gen(tokens + k)
    n = 300
    wp, ws = ref.weight(g, n, k)
    codes = ref.unpack(wp)
    codes[:, :32] = 0
    w = ref.pack(codes).contiguous()
    wd, wv = ops.Mxfp4Weight.from_checkpoint(w, ws), ref.values(codes, ws)
    for below in (20, 41, 60, 100):
        x = torch.randn(tokens, k, generator=g, device="cuda")
        x[:, 32:] *= 2.0 ** -below
        x[:, 1:32] = 0
        x[:, 0] = 1.0
        x = x.to(dtype)
        xv = x.double()
        want = xv @ wv.t()
        y = ops.Mxfp4DecodePlan(64, n, k).run(x, wd, out_dtype=torch.float32).double()
        assert want[:, :8].abs().amax() >= 2.0 ** (-below - 12)
        assert ((y - want).abs() <= block_bound(xv, wv, dtype)).all(), below


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens,k", [(1, 1024), (2, 1056), (4, 1024), (8, 1056), (16, 1056), (12, 1024)])
def test_decode_scales_at_the_ends_of_the_range(tokens, k, dtype):
    """Activations and weight scales that are huge on one side and tiny on the other: the products lie in f32's range, the scales' do not."""
    g = gen(tokens)
    n = 64
    codes = torch.randint(0, 16, (n, k), generator=g, device="cuda", dtype=torch.uint8)
    for x_exponent, w_exponent in ((120, -100), (-120, 100), (100, -127), (-100, 127), (60, 50), (-60, -50)):
        x = (torch.randn(tokens, k, generator=g, device="cuda") * 2.0 ** x_exponent).to(dtype)
        ws = torch.full((n, k // 32), 127 + w_exponent, dtype=torch.uint8, device="cuda")
        w = ops.Mxfp4Weight.from_checkpoint(ref.pack(codes).contiguous(), ws)
        xv, wv = x.double(), ref.values(codes, ws)
        y = ops.Mxfp4DecodePlan(64, n, k).run(x, w, out_dtype=torch.float32).double()
        assert ((y - xv @ wv.t()).abs() <= block_bound(xv, wv, dtype) + 2.0 ** -125 * (k // 32)).all(), (x_exponent, w_exponent)


@pytest.mark.parametrize("tokens,k,dtype", [(9, 1024, torch.bfloat16), (64, 1024, torch.bfloat16), (5, 1024, torch.float32), (1, 8192, torch.bfloat16)])
def test_decode_weights_aligned_to_16_bytes_only(tokens, k, dtype):
    """They take the other form of the product: other sums, the same bounds."""
    g = gen(24)
    n = 200
    wp, ws = ref.weight(g, n, k)
    buffer = torch.zeros(wp.numel() + 16, device="cuda", dtype=torch.uint8)
    odd = buffer[16:].view(n, k // 2)
    odd.copy_(wp)
    w = ops.Mxfp4Weight.from_checkpoint(odd, ws)
    assert w.packed.data_ptr() % 32 == 16
    x = randn(g, tokens, k, dtype=dtype)
    xv, wv = x.double(), ref.values(ref.unpack(wp), ws)
    plan = ops.Mxfp4DecodePlan(64, n, k)
    for weight in (w, ops.Mxfp4Weight.from_checkpoint(wp, ws)):
        y = plan.run(x, weight, out_dtype=torch.float32).double()
        assert ((y - xv @ wv.t()).abs() <= block_bound(xv, wv, dtype)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens,k", [(1, 1024), (3, 96), (6, 1056), (16, 544), (9, 1024), (24, 256), (64, 1024)])
def test_decode_results_at_the_end_of_the_range(tokens, k, dtype):
    """Results that f32 holds although a part of their sum, or an element rounded up, lies beyond it; and results that it does not hold."""
    g = gen(25)
    n = 40
    codes = torch.zeros(n, k, device="cuda", dtype=torch.uint8)
    codes[0, :3] = torch.tensor([2, 2, 10], device="cuda", dtype=torch.uint8)       # 1, 1, -1
    codes[1, 0] = 2                                                                # one element by itself
    codes[2, :2] = 2                                                               # overflows
    codes[3, :2] = 10
    codes[4, 0], codes[4, 40], codes[4, 41] = 2, 2, 10                             # over two blocks
    codes[5, 5:] = torch.randint(0, 16, (k - 5,), generator=g, device="cuda", dtype=torch.uint8)
    ws = torch.full((n, k // 32), 127, dtype=torch.uint8, device="cuda")
    x = randn(g, tokens, k)
    x[:, :3] = x[:, 40:42] = torch.finfo(dtype).max
    x = x.to(dtype)
    w = ops.Mxfp4Weight.from_checkpoint(ref.pack(codes).contiguous(), ws)
    xv, wv = x.double(), ref.values(codes, ws)
    want = (xv @ wv.t()).float()
    y = ops.Mxfp4DecodePlan(64, n, k).run(x, w, out_dtype=torch.float32)
    largest = torch.full_like(y[:, 0], float(torch.finfo(dtype).max))
    assert torch.equal(y[:, 0], largest) and torch.equal(y[:, 1], largest) and torch.equal(y[:, 4], largest)
    assert torch.equal(y[:, 2], torch.full_like(largest, float("inf"))) and torch.equal(y[:, 3], torch.full_like(largest, -float("inf")))
    assert not y[:, 6:].any() and torch.isfinite(want[:, 5]).sum() == torch.isfinite(y[:, 5]).sum()


@pytest.mark.parametrize("n,k,tokens,dtype", [(30001, 512, 5, torch.bfloat16), (60000, 512, 48, torch.bfloat16), (60000, 512, 64, torch.bfloat16), (30001, 512, 24, torch.float32),
                                              (60001, 2304, 1, torch.bfloat16)])
def test_decode_of_an_lm_head(n, k, tokens, dtype):
    """More row tiles than the device runs at a time: clusters of one CTA, several rounds of them, tensor memory handed on within an SM."""
    g = gen(26)
    x, w = randn(g, tokens, k, dtype=dtype), ops.Mxfp4Weight.from_checkpoint(*ref.weight(g, n, k))
    plan = ops.Mxfp4DecodePlan(64, n, k)
    y = plan.run(x, w, out_dtype=torch.float32)
    assert torch.equal(plan.run(x, w, out_dtype=torch.float32), y)
    xv = x.double()
    for first in range(0, n, 8192):
        wv = w.dequantize()[first: first + 8192].double()
        assert ((y[:, first: first + 8192].double() - xv @ wv.t()).abs() <= block_bound(xv, wv, dtype)).all()
    assert plan.status() == 0


@pytest.mark.parametrize("m,n", [(512, 5001), (1000, 5000), (1200, 1001), (520, 13), (2048, 1032)])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_gemm_ragged_outputs_on_cta_pairs(m, n, out):
    """Rows of the output that are no multiple of 16 elements, with beta * C, at 4, 8, 10, 5 and 16 row tiles."""
    g = gen(m)
    k = 544
    x = randn(g, m, k)
    xq, w = ops.quantize_mxfp4(x), ops.Mxfp4Weight.from_checkpoint(*ref.weight(g, n, k))
    xv, wv = ref.values(*ref.quantize(x)), w.dequantize().double()
    plan = ops.Mxfp4MatmulPlan(m, n, k)
    c = randn(g, m, n, dtype=out)
    want = xv @ wv.t() - 0.5 * c.double()
    bound = rounded(product_bound(xv, wv, 2) + 2.0 ** -23 * c.double().abs(), want, out)
    codes = [plan.block_n, 384, 512]
    for code in codes:
        plan.set_block_n(code)
        guarded = torch.full((m * n + 64,), 7.0, device="cuda", dtype=out)
        y = plan.run(xq, w, out=guarded[: m * n].view(m, n), beta=-0.5, c=c)
        assert ((y.double() - want).abs() <= bound).all(), code
        assert (guarded[m * n:] == 7.0).all()
    assert plan.status() == 0


def test_more_weights_than_a_plan_remembers():
    """A model's layers share a plan: twenty weights in turn, twice, and one whose memory is used again."""
    g = gen(27)
    n, k = 300, 512
    x = randn(g, 9, k, dtype=torch.bfloat16)
    weights = [ops.Mxfp4Weight.from_checkpoint(*ref.weight(g, n, k)) for _ in range(20)]
    decode, gemm, xq = ops.Mxfp4DecodePlan(16, n, k), ops.Mxfp4MatmulPlan(9, n, k), ops.quantize_mxfp4(x)
    first = [(ops.Mxfp4DecodePlan(16, n, k).run(x, w), ops.Mxfp4MatmulPlan(9, n, k).run(xq, w)) for w in weights]
    for _ in range(2):
        for w, (a, b) in zip(weights, first):
            assert torch.equal(decode.run(x, w), a) and torch.equal(gemm.run(xq, w), b)
    for part in ("packed", "scales_row_major", "scales_tiled", "scales_rows"):
        getattr(weights[0], part).copy_(getattr(weights[1], part))
    assert torch.equal(decode.run(x, weights[0]), first[1][0]) and torch.equal(gemm.run(xq, weights[0]), first[1][1])


def test_silu_quantizer_with_large_gates():
    """e^-gate is off by |gate| * 2^-23 of itself and vanishes below -87.3: a block of such gates keeps its codes but for boundaries, and
    what vanishes is below 2^-119 of up."""
    g = gen(28)
    rows, k = 256, 512
    gate = torch.linspace(-85, 85, rows, device="cuda").unsqueeze(1) + torch.randn(rows, k, generator=g, device="cuda")
    up = torch.randn(rows, k, generator=g, device="cuda")
    m = ops.silu_mul_halves_quantize_mxfp4(torch.cat([gate, up], 1))
    act = ref.silu_mul(torch.cat([gate, up], 1).double())
    codes, scales = ref.quantize(act)
    got, clean = ref.untile(m.scales, rows, k)
    assert clean
    # 95 * 2^-23 of a value, and about seven boundaries over a block's range: under 1e-4 of the codes
    assert (got != scales).float().mean() <= 1e-3 and (ref.unpack(m.packed) != codes).float().mean() <= 1e-3
    step = torch.exp2(scales.double() - 127).repeat_interleave(32, 1) * 2
    assert ((m.dequantize().double() - act).abs() <= step * 1.01).all()
    far = torch.cat([torch.full((4, 64), -95.0, device="cuda"), torch.full((4, 64), 3.0, device="cuda")], 1)
    far[1, :64], far[2, :64], far[3, :64] = -300.0, 90.0, 3e38
    far[3, 64:] = 0.5
    y = ops.silu_mul_halves_quantize_mxfp4(far).dequantize().double()
    assert y[:2].abs().max() <= 3 * 2.0 ** -119 and (y[2] == 256.0).all() and torch.isfinite(y[3]).all() and (y[3] >= 1e38).all()
    far[0, 0], far[1, 40], far[2, 0], far[3, 63] = float("nan"), float("inf"), -float("inf"), float("nan")
    y = ops.silu_mul_halves_quantize_mxfp4(far).dequantize()
    bad = torch.isnan(y)
    assert bad[0, :32].all() and bad[1, 32:].all() and bad[2, :32].all() and bad[3, 32:].all() and int(bad.sum()) == 4 * 32


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_poisoned_tokens_stay_alone_in_the_routed_layer(value):
    g = gen(29)
    tokens, experts, top_k, hidden, inter = 70, 8, 3, 160, 96
    gate_up, down = ([t.reshape(experts, -1, t.shape[1]) for t in ref.weight(g, experts * n, k, std=0.1)] for n, k in ((2 * inter, hidden), (hidden, inter)))
    gu, dn = ops.GroupedMxfp4Weights.from_checkpoint(*gate_up).interleave_gate_up(), ops.GroupedMxfp4Weights.from_checkpoint(*down)
    x, logits = randn(g, tokens, hidden), randn(g, tokens, experts)
    moe = ops.GroupedMoe(tokens, experts, top_k, hidden, inter, weight_format="mxfp4")
    clean = moe.run(x, logits, None, dn, w_gate_up_interleaved=gu).clone()
    x[11, 7], x[12, 159] = value, value
    y = moe.run(x, logits, None, dn, w_gate_up_interleaved=gu)
    others = torch.ones(tokens, dtype=torch.bool, device="cuda")
    others[11:13] = False
    assert torch.isnan(y[11:13]).all() and torch.equal(y[others], clean[others])
