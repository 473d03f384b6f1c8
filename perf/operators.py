"""MXFP4 linears (quantisation, products for many and few tokens, experts' products) and the selection step of beam search, as
cases to measure: each in a plain form of elementary torch operations, and through eider_b200.ops where `own` is true.

An MXFP4 block is 32 consecutive elements of a row: E2M1 codes (two to a byte, low nibble first) and one E8M0 scale byte c that
stands for 2^(c - 127).  A block's scale is 2^(floor(log2 amax) - 2), its codes are the elements over that scale, rounded to
nearest even and saturated at 6.

Layer sizes are those of the benchmark and of the test suite (hidden 5120 with an FFN of 13824, routed layers of 128 experts,
top-8, hidden 2048, expert intermediate 768); other sizes are generic ones around them.  Weights are N(0, 0.02^2), activations
and router logits N(0, 1).
"""
import math

import torch

own = False

LISTED = [
    # One token's activation on its way into a decode linear: the smallest call there is.
    {"name": "quantize_1", "kind": "quantize", "tokens": 1, "k": 5120, "dtype": "bf16"},
    # The largest chunk of the benchmark's sweep in front of the down projection.
    {"name": "quantize_16384", "kind": "quantize", "tokens": 16384, "k": 13824, "dtype": "bf16"},
    # The benchmark's prefill chunk through the fused gate/up projection, quantized on the fly.
    {"name": "linear_512", "kind": "linear", "tokens": 512, "k": 5120, "n": 27648, "dtype": "bf16", "out": "bf16"},
    # A ragged last chunk through a projection whose K ends inside a scale tile (2912 = 22.75 * 128), f32 in and out.
    {"name": "linear_333", "kind": "linear", "tokens": 333, "k": 2912, "n": 5000, "dtype": "f32", "out": "f32"},
    # The whole gated FFN of a 2048-token chunk with its residual.
    {"name": "ffn_2048", "kind": "ffn", "tokens": 2048, "hidden": 5120, "inter": 13824, "dtype": "bf16"},
    # One user's decode step: four up projections, each on its own activation and weights (more than the L2 holds).
    {"name": "decode_1", "kind": "decode", "tokens": 1, "k": 5120, "n": 13824, "layers": 4, "dtype": "bf16"},
    # A few sequences with f32 activations through a narrower layer with an odd number of outputs.
    {"name": "decode_5", "kind": "decode", "tokens": 5, "k": 4064, "n": 6150, "layers": 4, "dtype": "f32"},
    # A batch of 48 running sequences through the down projection.
    {"name": "decode_48", "kind": "decode", "tokens": 48, "k": 13824, "n": 5120, "layers": 4, "dtype": "bf16"},
    # The routed layer of the benchmark: 4096 tokens, 128 experts, top-8.
    {"name": "experts_4096", "kind": "experts", "tokens": 4096, "experts": 128, "top_k": 8, "hidden": 2048, "inter": 768, "dtype": "bf16"},
    # A short ragged prompt through the same layer: most experts see a handful of rows.
    {"name": "experts_77", "kind": "experts", "tokens": 77, "experts": 128, "top_k": 8, "hidden": 2048, "inter": 768, "dtype": "bf16"},
    # One request with four beams, f32 logits of a small vocabulary; the states are a short sequence's.
    {"name": "beam_1x4", "kind": "beam", "batch": 1, "beams": 4, "vocab": 32000, "k": 8, "dtype": "f32", "finished": 0.0, "state": 16384},
    # A full batch with eight beams each over a large vocabulary; some beams have ended.
    {"name": "beam_64x8", "kind": "beam", "batch": 64, "beams": 8, "vocab": 151936, "k": 16, "dtype": "bf16", "finished": 0.1, "state": 65536},
]


def listed():
    return [dict(c) for c in LISTED]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def _multiple(rng, lo, hi, step):
    return max(lo, min(hi, _log_int(rng, lo, hi) // step * step))


def draw(rng):
    """One more case: any kind, sizes spread over the range (over its logarithm), token counts of every residue."""
    kind = rng.choice(["quantize", "linear", "linear", "ffn", "decode", "decode", "experts", "beam", "beam"])
    if kind == "quantize":
        return {"kind": kind, "tokens": _log_int(rng, 1, 16384), "k": _multiple(rng, 64, 13824, 32), "dtype": rng.choice(["bf16", "f32"])}
    if kind == "linear":
        k, n = _multiple(rng, 512, 13824, 32), _log_int(rng, 256, 27648)
        n -= n % rng.choice([1, 8, 64, 128])
        return {"kind": kind, "tokens": _log_int(rng, 1, min(8192, 430_000_000_000 // (n * k))), "k": k, "n": n,
                "dtype": rng.choice(["bf16", "bf16", "f32"]), "out": rng.choice(["bf16", "bf16", "f32"])}
    if kind == "ffn":
        hidden, inter = rng.choice([(5120, 13824), (2048, 6144), (4096, 12288), (2880, 2880), (1024, 2784)])
        return {"kind": kind, "tokens": _log_int(rng, 1, 2048), "hidden": hidden, "inter": inter, "dtype": rng.choice(["bf16", "bf16", "f32"])}
    if kind == "decode":
        k = _multiple(rng, 512, 13824, 32)
        return {"kind": kind, "tokens": _log_int(rng, 1, 64), "k": k, "n": _log_int(rng, 256, min(13824, 13824 * 5120 // k)),
                "layers": 4, "dtype": rng.choice(["bf16", "bf16", "f32"])}
    if kind == "experts":
        return {"kind": kind, "tokens": _log_int(rng, 1, 4096), "experts": rng.choice([32, 64, 128]), "top_k": rng.choice([2, 4, 6, 8]),
                "hidden": rng.choice([1024, 2048, 2880]), "inter": rng.choice([512, 768, 1024]), "dtype": rng.choice(["bf16", "bf16", "f32"])}
    beams = rng.choice([1, 2, 3, 4, 5, 8, 16])
    batch = _log_int(rng, 1, 512 // beams)
    return {"kind": kind, "batch": batch, "beams": beams, "vocab": _log_int(rng, 1000, 151936), "k": beams * rng.choice([1, 2]),
            "dtype": rng.choice(["bf16", "f32"]) if batch * beams <= 256 else "bf16", "finished": rng.choice([0.0, 0.0, 0.2]),
            "state": 2 * _log_int(rng, 64, 32768)}


# ---- inputs ------------------------------------------------------------------------------------------------
_DTYPE = {"bf16": torch.bfloat16, "f32": torch.float32}


def _rng(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, shape, dtype=torch.float32, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).mul_(std).to(dtype)


def _weight(g, n, k):
    """A checkpoint's MXFP4 weight [n, k]: packed codes [n, k / 2] and scale bytes [n, k / 32] of N(0, 0.02^2) values."""
    packed, scales = [], []
    for rows in _normal(g, (n, k), std=0.02).split(8192):
        b = rows.reshape(rows.shape[0], -1, 32)
        exponent = torch.frexp(b.abs().amax(-1))[1] - 3
        a = (b * _pow2(-exponent)[..., None]).reshape(rows.shape)
        code = _code(a.abs()) | (a < 0).to(torch.uint8) << 3
        packed.append(code[:, 0::2] | code[:, 1::2] << 4)
        scales.append((exponent + 127).to(torch.uint8))
    return torch.cat(packed), torch.cat(scales)


def _pow2(exponent):
    """2^exponent in 32 bits, exactly."""
    return ((exponent.int() + 127) << 23).view(torch.float32)


def _code(a):
    """The E2M1 magnitude code nearest to a >= 0 (ties to the even code, 6 at most)."""
    return ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)).to(torch.uint8)


def _states(g, case):
    shape = (case["batch"], case["beams"], case["state"] // 2)
    return [_normal(g, shape, torch.bfloat16) for _ in range(2)]


def _beam_inputs(g, case):
    b, w, v = case["batch"], case["beams"], case["vocab"]
    logits = _normal(g, (b, w, v), std=2.5).to(_DTYPE[case["dtype"]])
    scores = torch.rand(b, w, generator=g, device="cuda").mul_(-8.0).sort(1, descending=True)[0]
    finished = torch.rand(b, w, generator=g, device="cuda") < case["finished"]
    return logits, scores, finished, _states(g, case)


def prepare(case, seed):
    g, kind = _rng(seed), case["kind"]
    state = {"case": dict(case)}
    if kind in ("quantize", "linear"):
        state["x"] = _normal(g, (case["tokens"], case["k"]), _DTYPE[case["dtype"]])
        if kind == "linear":
            state["w"] = _weight(g, case["n"], case["k"])
    elif kind == "decode":
        state["x"] = [_normal(g, (case["tokens"], case["k"]), _DTYPE[case["dtype"]]) for _ in range(case["layers"])]
        state["w"] = [_weight(g, case["n"], case["k"]) for _ in range(case["layers"])]
    elif kind == "ffn":
        t, h, i = case["tokens"], case["hidden"], case["inter"]
        state["w"] = [_weight(g, 2 * i, h), _weight(g, h, i)]
        state["x"], state["residual"] = _normal(g, (t, h), _DTYPE[case["dtype"]]), _normal(g, (t, h), torch.bfloat16)
    elif kind == "experts":
        t, e, h, i = case["tokens"], case["experts"], case["hidden"], case["inter"]
        # every expert's gate rows come before its up rows
        state["w"] = [[t.reshape(e, -1, t.shape[1]) for t in _weight(g, e * 2 * i, h)], [t.reshape(e, -1, t.shape[1]) for t in _weight(g, e * h, i)]]
        state["x"], state["logits"] = _normal(g, (t, h), _DTYPE[case["dtype"]]), _normal(g, (t, e))
    else:
        state["logits"], state["scores"], state["finished"], state["states"] = _beam_inputs(g, case)
    if own:
        _load(state)
    return state


def _load(state):
    """What a program makes of a checkpoint's weights when it loads them, and the plans it keeps."""
    from eider_b200 import ops
    case, kind = state["case"], state["case"]["kind"]
    if kind == "linear":
        state["weight"] = ops.Mxfp4Weight.from_checkpoint(*state["w"])
        state["plan"] = ops.Mxfp4MatmulPlan(case["tokens"], case["n"], case["k"])
    elif kind == "decode":
        state["weight"] = [ops.Mxfp4Weight.from_checkpoint(*w) for w in state["w"]]
        state["plan"] = ops.Mxfp4DecodePlan(case["tokens"], case["n"], case["k"])
    elif kind == "ffn":
        state["ffn"] = ops.DenseFfn(*[ops.Mxfp4Weight.from_checkpoint(*w) for w in state["w"]])
        state["ffn"].plans(case["tokens"])
    elif kind == "experts":
        state["weight"] = [ops.GroupedMxfp4Weights.from_checkpoint(*w) for w in state["w"]]
        state["interleaved"] = state["weight"][0].interleave_gate_up()
        state["moe"] = ops.GroupedMoe(case["tokens"], case["experts"], case["top_k"], case["hidden"], case["inter"], weight_format="mxfp4")


# ---- the plain forms, in 32 bits -----------------------------------------------------------------------------
def _rounded(x):
    """What the MXFP4 codes of x stand for (blocks of 32 along the last axis), exact in 32 bits."""
    b = x.float().reshape(-1, 32)
    amax = b.abs().amax(-1, keepdim=True)
    exponent = torch.where(amax > 0, torch.frexp(amax)[1] - 3, 0)
    a = b * _pow2(-exponent)
    code = _code(a.abs()).float()
    step = torch.where(code < 4, 0.5 * code, torch.where(code < 6, code - 2, 2 * code - 8))
    return (torch.copysign(step, b) * _pow2(exponent)).reshape(x.shape)


def _values(packed, scales):
    """The 32-bit values of packed codes [..., k / 2] with scale bytes [..., k / 32]."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=packed.device)
    code = torch.stack([packed & 15, packed >> 4], -1).reshape(-1).int()
    v = table.index_select(0, code).reshape(*scales.shape, 32)
    return (v * _pow2(scales.int() - 127)[..., None]).reshape(*packed.shape[:-1], -1)


def _silu_mul(gate_up):
    gate, up = gate_up.chunk(2, -1)
    return gate / (1.0 + torch.exp(-gate)) * up


def _experts(state):
    case, x, logits = state["case"], state["x"], state["logits"]
    t, e, s = case["tokens"], case["experts"], case["top_k"]
    top, chosen = logits.topk(s, 1)
    top = torch.exp(top - top[:, :1])
    weight = (top / top.sum(1, keepdim=True)).reshape(-1)
    chosen = chosen.reshape(-1)
    order = chosen.argsort(stable=True)
    counts = torch.bincount(chosen, minlength=e)
    first = counts.cumsum(0) - counts
    expert = chosen[order]
    place = expert, torch.arange(t * s, device=x.device) - first[expert]  # the route's row among its expert's
    rows = torch.zeros(e, int(counts.max()), case["hidden"], device=x.device)
    rows[place] = _rounded(x)[order // s]
    act = _silu_mul(torch.bmm(rows, _values(*state["w"][0]).transpose(1, 2)))
    down = torch.bmm(_rounded(act), _values(*state["w"][1]).transpose(1, 2))[place]
    back = torch.empty_like(down)
    back[order] = down * weight[order, None]
    return back.reshape(t, s, -1).sum(1).to(torch.bfloat16)


def _beam(state):
    case, logits = state["case"], state["logits"].double()
    b, w, v = logits.shape
    top = logits.amax(-1, keepdim=True)
    score = logits - top - torch.log(torch.exp(logits - top).sum(-1, keepdim=True)) + state["scores"].double()[..., None]
    score = torch.where(state["finished"][..., None], -math.inf, score)
    score[..., 0] = torch.where(state["finished"], state["scores"].double(), score[..., 0])  # token 0 is the padding token
    best, at = score.reshape(b, w * v).sort(dim=1, descending=True, stable=True)
    best, at = best[:, : case["k"]], at[:, : case["k"]]
    parents, tokens = torch.div(at, v, rounding_mode="floor"), at % v
    batch = torch.arange(b, device=at.device)[:, None]
    return {"scores": best.float(), "parents": parents.int(), "tokens": tokens.int(), "states": [s[batch, parents[:, :w]] for s in state["states"]]}


def run(state):
    case, kind = state["case"], state["case"]["kind"]
    if own:
        return _own(state, case, kind)
    if kind == "quantize":
        return _rounded(state["x"]).to(state["x"].dtype)
    if kind == "linear":
        return (_rounded(state["x"]) @ _values(*state["w"]).t()).to(_DTYPE[case["out"]])
    if kind == "decode":
        return [(x.float() @ _values(*w).t()).to(x.dtype) for x, w in zip(state["x"], state["w"])]
    if kind == "ffn":
        gate_up, down = state["w"]
        act = _silu_mul(_rounded(state["x"]) @ _values(*gate_up).t())
        return (_rounded(act) @ _values(*down).t() + state["residual"].float()).to(torch.bfloat16)
    return _experts(state) if kind == "experts" else _beam(state)


def _own(state, case, kind):
    from eider_b200 import ops
    if kind == "quantize":
        return ops.quantize_mxfp4(state["x"]).dequantize(state["x"].dtype)
    if kind == "linear":
        return state["plan"].run(ops.quantize_mxfp4(state["x"]), state["weight"], out_dtype=_DTYPE[case["out"]])
    if kind == "decode":
        plan = state["plan"]
        return [plan.run(x, w, out_dtype=x.dtype) for x, w in zip(state["x"], state["weight"])]
    if kind == "ffn":
        return state["ffn"].run(state["x"], state["residual"])
    if kind == "experts":
        return state["moe"].run(state["x"], state["logits"], state["weight"][0], state["weight"][1], w_gate_up_interleaved=state["interleaved"],
                                out_dtype=torch.bfloat16)
    scores, parents, tokens = ops.beam_search_select(state["logits"], state["scores"], case["k"], finished=state["finished"], pad_token=0)
    return {"scores": scores, "parents": parents, "tokens": tokens, "states": ops.beam_search_reorder(state["states"], parents[:, : case["beams"]])}


# ---- the same results in 64 bits ----------------------------------------------------------------------------
_GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _exact_rounded(x):
    """Block scale and nearest grid value in 64 bits: the two neighbours of each element are looked up and the nearer one taken."""
    parts = []
    grid = torch.tensor(_GRID, dtype=torch.float64, device=x.device)
    for rows in x.double().split(4096):
        b = rows.reshape(rows.shape[0], -1, 32)
        largest = b.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -125)
        scale = 0.125 * largest / torch.frexp(largest)[0]  # the power of two two places below the largest element's
        a = (b / scale).abs().clamp(max=6.0)
        above = torch.searchsorted(grid, a).clamp(1, 7)
        low, high = grid[above - 1], grid[above]
        up = (a - low > high - a) | ((a - low == high - a) & (above % 2 == 0))
        parts.append((torch.where(up, high, low) * b.sign() * scale).reshape(rows.shape))
    return torch.cat(parts)


def _exact_values(packed, scales):
    """A weight's values in 64 bits, half the columns from each nibble."""
    grid = torch.tensor(_GRID, dtype=torch.float64, device=packed.device)
    out = torch.empty(packed.shape[0], 2 * packed.shape[1], dtype=torch.float64, device=packed.device)
    for first, nibble in ((0, packed % 16), (1, packed // 16)):
        out[:, first::2] = grid[(nibble % 8).long()] * (1.0 - 2.0 * (nibble // 8).double())
    return out * torch.ldexp(torch.ones_like(scales, dtype=torch.float64), scales.int() - 127).repeat_interleave(32, 1)


def _exact_times(x, w):
    """x . w^T of a checkpoint's weight, a slab of it at a time."""
    return torch.cat([x @ _exact_values(p, s).t() for p, s in zip(w[0].split(4096), w[1].split(4096))], 1)


def _exact_act(gate_up):
    half = gate_up.shape[1] // 2
    return gate_up[:, :half] * torch.sigmoid(gate_up[:, :half]) * gate_up[:, half:]


def exact(case, seed):
    """The results of `run` from the same inputs, every product and sum in 64 bits; only what the path holds in MXFP4 is rounded
    to it here too."""
    g, kind = _rng(seed), case["kind"]
    if kind == "beam":
        logits, scores, finished, states = _beam_inputs(g, case)
        b, w, v = logits.shape
        total = torch.log_softmax(logits.double(), -1) + scores.double().unsqueeze(-1)
        total[finished] = -math.inf
        total[..., 0][finished] = scores.double()[finished]
        best = total.reshape(b, -1).topk(case["k"], 1)[0]
        # parents and tokens are whole numbers, and the states move by them
        return {"scores": best, "parents": None, "tokens": None, "states": [None, None]}
    if kind in ("quantize", "linear"):
        x = _exact_rounded(_normal(g, (case["tokens"], case["k"]), _DTYPE[case["dtype"]]))
        return x if kind == "quantize" else _exact_times(x, _weight(g, case["n"], case["k"]))
    if kind == "decode":
        xs = [_normal(g, (case["tokens"], case["k"]), _DTYPE[case["dtype"]]).double() for _ in range(case["layers"])]
        return [_exact_times(x, _weight(g, case["n"], case["k"])) for x in xs]
    t, h, i = case["tokens"], case["hidden"], case["inter"]
    if kind == "ffn":
        gate_up, down = _weight(g, 2 * i, h), _weight(g, h, i)
        x, residual = _normal(g, (t, h), _DTYPE[case["dtype"]]), _normal(g, (t, h), torch.bfloat16)
        act = _exact_act(_exact_times(_exact_rounded(x), gate_up))
        return _exact_times(_exact_rounded(act), down) + residual.double()
    e = case["experts"]
    gate_up, down = [[p.reshape(e, -1, p.shape[1]) for p in _weight(g, e * n, k)] for n, k in ((2 * i, h), (h, i))]
    x, logits = _normal(g, (t, h), _DTYPE[case["dtype"]]), _normal(g, (t, e))
    top, chosen = logits.double().topk(case["top_k"], 1)
    weights, xq, out = torch.softmax(top, 1), _exact_rounded(x), torch.zeros(t, h, dtype=torch.float64, device="cuda")
    for c in range(e):
        rows, slot = (chosen == c).nonzero(as_tuple=True)
        if len(rows):
            act = _exact_act(_exact_times(xq[rows], (gate_up[0][c], gate_up[1][c])))
            out[rows] += weights[rows, slot, None] * _exact_times(_exact_rounded(act), (down[0][c], down[1][c]))
    return out


def work(case):
    """Every input read once, every output written once; MXFP4 takes 17/32 byte an element."""
    kind, size = case["kind"], {"bf16": 2, "f32": 4}
    if kind == "quantize":
        return {"bytes": 2 * case["tokens"] * case["k"] * size[case["dtype"]], "flops": 0}
    if kind == "linear":
        t, k, n = case["tokens"], case["k"], case["n"]
        return {"bytes": n * k * 17 // 32 + t * k * size[case["dtype"]] + t * n * size[case["out"]], "flops": 2 * t * n * k}
    if kind == "decode":
        t, k, n, b = case["tokens"], case["k"], case["n"], size[case["dtype"]]
        return {"bytes": case["layers"] * (n * k * 17 // 32 + t * (k + n) * b), "flops": case["layers"] * 2 * t * n * k}
    if kind == "ffn":
        t, h, i = case["tokens"], case["hidden"], case["inter"]
        return {"bytes": 3 * h * i * 17 // 32 + t * h * (size[case["dtype"]] + 4), "flops": 6 * t * h * i}
    if kind == "experts":
        t, e, s, h, i = case["tokens"], case["experts"], case["top_k"], case["hidden"], case["inter"]
        touched = e * (1.0 - (1.0 - s / e) ** t)  # experts that some token chose
        return {"bytes": int(touched * 3 * h * i * 17 / 32) + t * (h * (size[case["dtype"]] + 2) + 4 * e), "flops": 6 * t * s * h * i}
    rows = case["batch"] * case["beams"]
    return {"bytes": int(rows * (case["vocab"] * size[case["dtype"]] * (1.0 - case["finished"]) + 4 * case["state"])) + case["batch"] * case["k"] * 12,
            "flops": 4 * rows * case["vocab"]}
