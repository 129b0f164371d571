"""The oracle's quantized writes into blocks whose scale a program wrote itself, by hand."""
import math

import pytest
import torch

from oracle import cache8_oracle as CO


@pytest.mark.parametrize("codes,top", [(torch.int8, 127.0), (torch.float8_e4m3fn, 448.0)])
@pytest.mark.parametrize("was,now", [(-5.0, 5.0), (5.0, 5.0), (-0.5, 1.0), (0.5, 1.0), (0.0, 1.0), (-0.0, 1.0), (math.inf, math.inf), (-math.inf, -math.inf), (math.nan, math.nan)])
def test_scales_that_are_held(codes, top, was, now):
    """A row that asks for 1 goes to the second place of a block; what the first place holds keeps its value, as nearly as a code can."""
    held = torch.zeros(1, 1, 4, 16)
    held[0, 0, 0, :4] = torch.tensor([top, -top, 24.0, 0.0])
    cache, scale = held.to(codes), torch.full((1, 1, 1), was)
    row = torch.full((1, 1, 16), -top)
    kc, vc, ks, _ = CO.append(row, row, cache, cache, torch.tensor([1]), scale, scale)
    assert str(float(ks)) == str(now)
    if math.isfinite(now):
        assert CO.values(kc, ks)[0, 0, 0, :4].tolist() == pytest.approx((held[0, 0, 0, :4] * was).tolist(), rel=0, abs=now / 2 if codes == torch.int8 else top * now / 28)
        assert (CO.values(kc, ks)[0, 1, 0] + top).abs().max() <= (now / 2 if codes == torch.int8 else top * now / 28)
    else:
        assert torch.equal(CO.numbers(kc)[0, 0, 0], held[0, 0, 0].double()) and not CO.numbers(kc)[0, 0, 1].any()
