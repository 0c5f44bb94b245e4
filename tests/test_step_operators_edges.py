"""Calls of the operators of short ragged steps that are easily answered wrongly, on the CPU: what they refuse, and what the plain forms say."""
import pytest
import torch

from lorax_b200.ops import native, reference
from tests.test_step_operators import BF16, _moe_args, _refused, ints


# ------------------------------------------------------------------------------------------------ experts
def test_experts_refuse_a_result_on_top_of_their_inputs():
    """Tokens are routed by every block of the second kernel too, while others write."""
    a = _moe_args(T=4)
    rows = torch.zeros(8, 64, dtype=BF16)
    for over in (dict(out=a["x"]), dict(out=a["router_w"]), dict(out=a["w13"][1, :4]), dict(out=a["w2"].view(-1)[64:320].view(4, 64)),
                 dict(x=rows[:4], out=rows[3:7]), dict(x=rows[4:], out=rows[1:5]), dict(x=rows[0:8:2], out=rows[0:8:2]),
                 dict(x=torch.zeros(4, 128, dtype=BF16)[:, :64])):
        args = {**a, **over}
        if "out" not in over:
            args["out"] = args["x"].as_strided((4, 64), (128, 1), 32)
        with_out = dict(args)
        _refused("moe_few", **with_out)


def test_experts_into_a_result_between_the_rows_of_their_inputs():
    """Rows that take turns share nothing: such a result is written as any other."""
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g)
    wr, w13, w2 = r(4, 64), r(4, 64, 64), r(4, 64, 32)
    buf = torch.zeros(4, 128)
    buf[:, :64] = r(4, 64)
    want = reference.moe_few(buf[:, :64].clone(), wr, w13, w2, 2)
    got = reference.moe_few(buf[:, :64], wr, w13, w2, 2, out=buf[:, 64:])
    assert torch.equal(got, want) and torch.equal(buf[:, 64:], want)
    lines = torch.zeros(8, 64)
    lines[::2] = buf[:, :64]
    assert torch.equal(reference.moe_few(lines[::2], wr, w13, w2, 2, out=lines[1::2]), want)
