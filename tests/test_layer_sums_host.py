"""That the whole numbers of the tests of sums show a mistake: sixteen rows left out, or counted twice, change every gradient over the
rows, wherever they lie.  The mistake is in the oracle, on the CPU."""
import pytest
import torch

import whole_layers as W


def seen(total, part):
    for dtype in (torch.float16, torch.bfloat16):
        right = total.to(dtype)
        for wrong in (total - part, total + part):
            assert float((wrong.to(dtype) != right).float().mean()) > 0.05


@pytest.mark.parametrize("m,k,n", W.NARROW + [s for s in W.LARGE if s[0] * s[1] * s[2] < 1 << 33])
def test_lost_rows_of_a_linear_layer_show(m, k, n):
    x, w, b, r, dy = W.linear(m, k, n, "cpu")
    for relu in (False, True):
        _, _, dz = W.linear_want(x, w, b, r, dy, relu)
        gw, gb = torch.mm(dz.t().contiguous(), x.float()), dz.sum(0)
        for at in (0, m // 2 // 16 * 16, m - 16):
            seen(gw, torch.mm(dz[at:at + 16].t().contiguous(), x[at:at + 16].float()))
            seen(gb, dz[at:at + 16].sum(0))


@pytest.mark.parametrize("m,k", W.NORMS[:6])
def test_lost_rows_of_a_norm_show(m, k):
    x, dy, _ = W.norm(m, k, "cpu")
    dw = dy.float() * (x.float() / 2)
    total = dw.sum(0)
    for at in (0, m // 2, m - 1):
        seen(total, dw[at:at + 1].sum(0))
