"""Launches without a pause between them: each reads what the one in front of it has just written into a buffer that both turns use."""
import pytest
import torch

from eider_b200 import ops
from tests.util import require_cuda

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _cuda():
    require_cuda()


def consumers(tokens, k, n, g):
    """name -> what is computed from x, a list of tensors."""
    weight = torch.randn(n, k, generator=g, device="cuda") * 0.02
    nv, mx = ops.ModelOptWeight.quantize(weight), ops.Mxfp4Weight.quantize(weight)
    fp8, channel = ops.quantize_fp8_weight(weight)
    nv_decode, fp8_decode, mx_decode = ops.Nvfp4DecodePlan(64, n, k), ops.Fp8DecodePlan(64, n, k), ops.Mxfp4DecodePlan(64, n, k)
    nv_gemm, mx_gemm = ops.Fp4TnMatmulPlan(tokens, n, k), ops.Mxfp4MatmulPlan(tokens, n, k)
    routes = ops.MoeSortedRoutes(2 * tokens, 4)
    routes.sort(torch.randint(0, 4, (2 * tokens,), generator=g, device="cuda", dtype=torch.int32))
    nv_rows, mx_rows = ops.MoeSortedNvfp4Rows(2 * tokens, 4, k, tokens), ops.MoeSortedMxfp4Rows(2 * tokens, 4, k)

    def quantized(m):
        return [m.packed, m.scales] + ([m.row_scales] if getattr(m, "row_scales", None) is not None else [])

    def sorted_rows(rows, call):
        call()
        return [rows.packed.clone(), rows.scales.clone()]

    return {
        "nvfp4": lambda x: quantized(ops.quantize_nvfp4(x, 0.5)),
        "nvfp4 rows": lambda x: quantized(ops.quantize_nvfp4_rowscale(x)),
        "nvfp4 gemm": lambda x: [nv_gemm.run(ops.quantize_nvfp4_rowscale(x), nv)],
        "nvfp4 decode": lambda x: [nv_decode.run(x, nv)],
        "nvfp4 routes": lambda x: sorted_rows(nv_rows, lambda: nv_rows.gather_quantize(x, routes, 2)),
        "fp8 rows": lambda x: list(ops.quantize_fp8_dynamic(x)),
        "fp8 decode": lambda x: [fp8_decode.run(x, fp8, channel)],
        "mxfp4": lambda x: quantized(ops.quantize_mxfp4(x)),
        "mxfp4 gemm": lambda x: [mx_gemm.run(ops.quantize_mxfp4(x), mx)],
        "mxfp4 decode": lambda x: [mx_decode.run(x, mx)],
        "mxfp4 routes": lambda x: sorted_rows(mx_rows, lambda: mx_rows.quantize_routes(x, routes, 2)),
    }


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens,k,n", [(1, 512, 256), (3, 2048, 640), (40, 1024, 384)])
def test_consumers_read_what_the_combine_wrote(tokens, k, n, dtype):
    g = torch.Generator(device="cuda").manual_seed(tokens)
    order = ops.MoeSortedRoutes(tokens, 1)
    order.route_to_sorted.copy_(torch.arange(tokens, device="cuda", dtype=torch.int32))
    ones = torch.ones(tokens, device="cuda")
    rows = [torch.randn(tokens, k, generator=g, device="cuda").bfloat16() for _ in range(2)]
    x = torch.empty(tokens, k, device="cuda", dtype=dtype)
    for name, use in consumers(tokens, k, n, g).items():
        want = []
        for r in rows:
            x.copy_(r)
            torch.cuda.synchronize()
            want.append([t.clone() for t in use(x)])
            torch.cuda.synchronize()
        wrong = torch.zeros((), device="cuda", dtype=torch.int64)
        for i in range(60):
            ops.moe_weighted_accumulate(order, ones, rows[i % 2], tokens, 1, out=x)
            for got, expected in zip(use(x), want[i % 2]):
                wrong += (got != expected).any().long()
        assert int(wrong) == 0, name
