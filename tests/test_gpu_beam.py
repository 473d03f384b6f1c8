"""Beam search selection and reordering against a stable sort in 64 bits."""
import math

import pytest
import torch

from eider_b200 import ops
from tests import mxfp4_reference as ref
from tests.util import require_cuda

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _cuda():
    require_cuda()


def reference(logits, scores, k, finished=None, pad=0):
    """(scores in 64 bits, parents, tokens) from the definition."""
    b, w, v = logits.shape
    x, s = logits.double(), scores.double().unsqueeze(-1)
    top = x.amax(-1, keepdim=True)
    total = x - top - torch.log(torch.exp(x - top).sum(-1, keepdim=True)) + s  # (top apart: at 3e38 a sum with it loses the rest)
    dead = ~torch.isfinite(torch.logsumexp(x, -1, keepdim=True)) | ~torch.isfinite(s)
    total = torch.where(dead, -math.inf, total)
    if finished is not None:
        ended = finished.bool().unsqueeze(-1)
        total = torch.where(ended, -math.inf, total)
        total[..., pad] = torch.where(ended[..., 0] & torch.isfinite(s[..., 0]), s[..., 0], total[..., pad])
    best, at = total.reshape(b, w * v).sort(dim=1, descending=True, stable=True)
    return best[:, :k], at[:, :k] // v, at[:, :k] % v


def check(logits, scores, k, finished=None, pad=0):
    got, parents, tokens = ops.beam_search_select(logits, scores, k, finished=finished, pad_token=pad)
    want, p, t = reference(logits, scores, k, finished, pad)
    assert torch.equal(parents.long(), p) and torch.equal(tokens.long(), t)
    # a sum of exponentials within 2^-21 (hardware exponentials, f32 partial sums), one rounding to f32
    fine = torch.isfinite(want.float())
    assert torch.equal(torch.isfinite(got), fine)
    assert ((got.double() - want).abs()[fine] <= 2.0 ** -21 + 2.0 ** -24 * want.abs()[fine]).all()


def inputs(seed, b, w, v, dtype, std=2.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    logits = (torch.randn(b, w, v, generator=g, device="cuda") * std).to(dtype)
    return logits, -8 * torch.rand(b, w, generator=g, device="cuda"), g


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,w,v,k", [(1, 1, 1, 1), (1, 1, 7, 7), (2, 3, 5, 15), (1, 4, 32000, 8), (3, 5, 1001, 10), (7, 2, 4099, 4), (2, 16, 50257, 32),
                                     (1, 64, 640, 128), (40, 8, 3001, 16), (1, 2, 131072, 64)])
def test_select(b, w, v, k, dtype):
    logits, scores, _ = inputs(v + k, b, w, v, dtype)
    check(logits, scores, k)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_ties_go_to_the_lowest_index(dtype):
    logits, scores, g = inputs(1, 4, 4, 5000, dtype)
    logits = (logits.float() * 2).round().div(2).to(dtype)  # few values: long runs of equal ones
    check(logits, scores, 16)
    logits[:, 1:] = logits[:, :1]  # equal beams
    check(logits, scores[:, :1].expand(4, 4).contiguous(), 128)
    check(torch.zeros_like(logits), torch.zeros_like(scores), 100)  # one run: 20000 equal scores
    logits[0] = -0.0
    logits[0, :, ::3] = 0.0
    check(logits, torch.zeros_like(scores), 20)
    # one thread's worth of equal scores beyond what a selection ranks
    flat = torch.full((1, 2, 131072), -30.0, device="cuda", dtype=dtype)
    flat[0, 0, ::64] = 1.0
    check(flat, torch.zeros(1, 2, device="cuda"), 70)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masked_and_poisoned_rows(dtype):
    logits, scores, g = inputs(2, 6, 3, 900, dtype)
    logits[0, 0, 10:] = -math.inf            # few tokens left
    logits[0, 1:] = -math.inf                # nothing left
    logits[1, 1, 5] = math.nan
    logits[1, 2, 899] = math.inf
    logits[2] = -math.inf
    scores[3, 1:] = -math.inf                # the first step: one live beam
    scores[4, 0] = math.nan
    scores[5, 2] = math.inf
    logits[5, 0] = torch.finfo(dtype).min    # masks of the type's lowest value
    logits[5, 1, 7:] = torch.finfo(dtype).min
    for k in (1, 6, 40):
        check(logits, scores, k)
    huge = logits.clone()
    huge[0, 0, :10] = torch.linspace(-3e38, 3e38, 10, device="cuda").to(dtype)
    check(huge, scores, 12)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_finished_beams(dtype):
    logits, scores, g = inputs(3, 8, 4, 2001, dtype)
    finished = torch.rand(8, 4, generator=g, device="cuda") < 0.5
    finished[0], finished[1] = True, False
    scores[2, 0], finished[2, 0] = -math.inf, True
    logits[finished] = math.nan  # what a finished row holds does not matter
    for pad in (0, 1500, 2000):
        check(logits, scores, 8, finished, pad)
        check(logits, scores, 8, finished.to(torch.uint8), pad)
    check(logits[:1], scores[:1], 20, finished[:1], 3)  # four candidates for twenty places


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_apart_and_unaligned(dtype):
    logits, scores, _ = inputs(4, 3, 4, 3011, dtype)
    for v, first in ((3011, 0), (2999, 0), (2999, 1), (1000, 3), (64, 5), (3, 7)):
        check(logits[:, :, first: first + v], scores, 3)
    one = logits[1:2, 2:3, 5:800]
    check(one, scores[1:2, 2:3].contiguous(), 5)


def test_reorder():
    g = torch.Generator(device="cuda").manual_seed(5)
    for b, w in ((1, 1), (3, 4), (5, 8), (2, 64)):
        states = [torch.randn(b, w, 2, 130, generator=g, device="cuda"), torch.randint(0, 99, (b, w, 7), generator=g, device="cuda", dtype=torch.uint8),
                  torch.randn(b, w, 9001, generator=g, device="cuda").to(torch.bfloat16), torch.arange(b * w, device="cuda").reshape(b, w)]
        parents = torch.randint(0, w, (b, 2 * w), generator=g, device="cuda", dtype=torch.int32)[:, :w]
        got = ops.beam_search_reorder(states, parents)
        batch = torch.arange(b, device="cuda")[:, None]
        for s, o in zip(states, got):
            assert torch.equal(o, s[batch, parents.long()])
        # many states, into given outputs, whose rows without a parent stay as they are
        many = [states[0] + i for i in range(30)]
        out = [torch.full_like(t, -1) for t in many]
        wild = parents.clone()
        wild[0, 0] = w
        wild[-1, -1] = -1
        ops.beam_search_reorder(many, wild, out=out)
        keep = ((wild >= 0) & (wild < w))[..., None, None]
        for s, o in zip(many, out):
            assert torch.equal(o, torch.where(keep, s[batch, wild.clamp(0, w - 1).long()], torch.full_like(s, -1)))


def test_refusals():
    logits, scores, _ = inputs(6, 2, 4, 100, torch.float32)
    for bad in ({"logits": logits.half()}, {"logits": logits[0]}, {"logits": logits[:, :, ::2]}, {"logits": logits.transpose(0, 1)}, {"beam_scores": scores[:1]},
                {"beam_scores": scores.double()}, {"k": 0}, {"k": 129}, {"finished": scores}, {"finished": torch.zeros(2, 4, device="cuda", dtype=torch.bool), "pad_token": 100}):
        with pytest.raises(ops.ShapeError):
            ops.beam_search_select(**({"logits": logits, "beam_scores": scores, "k": 8} | bad))
    parents = torch.zeros(2, 4, device="cuda", dtype=torch.int32)
    state = torch.zeros(2, 4, 8, device="cuda")
    for args in (([], parents), ([state], parents.long()), ([state[:, :2]], parents), ([state.transpose(1, 2)], parents), ([state], parents, [state]),
                 ([state], parents, [torch.zeros(2, 4, 9, device="cuda")])):
        with pytest.raises(ops.ShapeError):
            ops.beam_search_reorder(*args)


def test_decode_steps_with_beams():
    """A few steps as a decode loop runs them: the MXFP4 lm-head over the beams' hidden states, selection, reordering of states, all in
    one captured graph on a stream of its own; every step against 64 bits from the same inputs."""
    g = torch.Generator(device="cuda").manual_seed(7)
    batch, beams, hidden, vocab = 3, 4, 512, 5003
    head = ops.Mxfp4Weight.from_checkpoint(*ref.weight(g, vocab, hidden, std=0.1))
    plan = ops.Mxfp4DecodePlan(batch * beams, vocab, hidden)
    x = torch.zeros(batch, beams, hidden, device="cuda", dtype=torch.bfloat16)
    scores = torch.zeros(batch, beams, device="cuda")
    states = [torch.randn(batch, beams, 3, 65, generator=g, device="cuda"), torch.randint(0, 9, (batch, beams, 40), generator=g, device="cuda")]

    def step():
        logits = plan.run(x.reshape(batch * beams, hidden), head, out_dtype=torch.float32).reshape(batch, beams, vocab)
        best, parents, tokens = ops.beam_search_select(logits, scores, 2 * beams)
        return best, parents, tokens, ops.beam_search_reorder(states, parents[:, :beams])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        best, parents, tokens, moved = step()
    scores[:, 1:] = -math.inf  # the first step has one beam
    wv = head.dequantize().double()
    for _ in range(4):
        x.copy_(torch.randn(batch, beams, hidden, generator=g, device="cuda"))
        before, started = [s.clone() for s in states], scores.clone()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.current_stream().wait_stream(side)
        want, p, t = reference((x.double() @ wv.t()), started, 2 * beams)
        assert torch.equal(parents.long(), p) and torch.equal(tokens.long(), t)
        assert (best.double() - want).abs().max() <= 1e-4
        for s, o in zip(before, moved):
            assert torch.equal(o, s[torch.arange(batch, device="cuda")[:, None], p[:, :beams]])
        scores.copy_(best[:, :beams])
        for s, o in zip(states, moved):
            s.copy_(o)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", [9, 67, 4099, 9001, 50257, 131071])
def test_equal_beams_tie_wherever_their_rows_lie(v, dtype):
    """Rows of an odd length start at every offset from a 16-byte boundary: the same logits give the same scores there, bit for bit, so equal
    beams come in the order of their index, and one candidate of every beam precedes the next token's."""
    b, w, k = 2, 16, min(16 * v, 100)
    logits, scores, g = inputs(v, b, 1, v, dtype)
    # (one row's scores in 64 bits: sums of w copies of it need not agree to the last bit there)
    top = logits.double().amax(-1, keepdim=True)
    total = logits.double() - top - torch.log(torch.exp(logits.double() - top).sum(-1, keepdim=True)) + scores.double().unsqueeze(-1)
    at = total.expand(b, w, v).reshape(b, w * v).sort(dim=1, descending=True, stable=True)[1][:, :k]
    logits = logits.expand(b, w, v).contiguous()
    _, parents, tokens = ops.beam_search_select(logits, scores.expand(b, w).contiguous(), k)
    assert torch.equal(parents.long(), at // v) and torch.equal(tokens.long(), at % v)
    got, parents, _ = ops.beam_search_select(logits, scores.expand(b, w).contiguous(), 16)
    assert torch.equal(parents, torch.arange(16, device="cuda", dtype=torch.int32).expand(b, 16)) and (got == got[:, :1]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", [1, 7, 8, 1000, 8196, 32003, 131072])
def test_scores_do_not_depend_on_alignment(v, dtype):
    b, w, k = 2, 3, min(3 * v, 64)
    logits, scores, g = inputs(v, b, w, v, dtype)
    want = ops.beam_search_select(logits, scores, k)
    for pitch, first in ((v + 8, 0), (v + 1, 0), (v + 1, 1), (v + 5, 3), (v + 8, 7), (v + 14, 5)):
        wide = torch.full((b, w, pitch), math.nan, device="cuda", dtype=dtype)
        copy = wide[:, :, first: first + v]
        copy.copy_(logits)
        for x, y in zip(ops.beam_search_select(copy, scores, k), want):
            assert torch.equal(x, y), (pitch, first)


@pytest.mark.parametrize("row_bytes", [65536, 65552, 300001, 8 << 20])
def test_reorder_long_states(row_bytes):
    """Rows beyond what one CTA copies at a time, as of key and value caches."""
    g = torch.Generator(device="cuda").manual_seed(9)
    b, w = (1, 4) if row_bytes > 1 << 20 else (3, 5)
    states = [torch.randint(0, 256, (b, w, row_bytes), generator=g, device="cuda", dtype=torch.uint8) for _ in range(2)]
    parents = torch.randint(0, w, (b, w), generator=g, device="cuda", dtype=torch.int32)
    batch = torch.arange(b, device="cuda")[:, None]
    for s, o in zip(states, ops.beam_search_reorder(states, parents)):
        assert torch.equal(o, s[batch, parents.long()])
