"""The decode step's operators at the edges of what their definitions allow, against plain
implementations in 64 bits: temperatures far from one, values at the ends of their types, NaN that
some rows see and others do not, bits lost on the way."""

import math

import pytest
import torch

from newt_b200 import ops
from newt_b200.runtime import abi
from test_decode_ops_gpu import BF16, FP16, FP32, HALF, _gen, _randn, _score_exact

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_kernel_gave_up():
    yield
    torch.cuda.synchronize()
    assert abi.read_status() == (0, 0)


def _agree(got, want, relative, floor):
    """|got - want| <= relative * |want| + floor where `want` is finite; elsewhere the same infinity,
    or NaN in both."""
    got, want = got.double(), want.double()
    finite = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf])
    off = (got - want).abs()[finite] - (relative * want.abs()[finite] + floor)
    worst = off.max().item() if off.numel() else 0.0
    assert worst <= 0.0, worst


# ---- log probabilities -------------------------------------------------------------------------

@pytest.mark.parametrize("inv", [1e-20, 1e-3, 0.1, 0.25, 0.5, 0.7, 0.9, 1.3, 1.7, 1e3, 1e6, 1e9, 1e20])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("rows, vocab, top", [(3, 1003, 5), (301, 1003, 5), (2, 40009, 0), (650, 33, 32)])
def test_token_logprobs_at_far_temperatures(rows, vocab, top, dtype, inv):
    """Masked and missing elements weigh nothing at any temperature, and the largest logit's rounding
    does not leave the range of an exponential."""
    gen = _gen(rows + vocab)
    x = _randn(gen, rows, vocab, dtype=dtype, scale=3.0)
    x[:, vocab - 7:] = -math.inf
    x[0, :vocab - 7:3] = torch.finfo(dtype).min
    tokens = 1 + 3 * torch.randint(0, (vocab - 8) // 3, (rows,), generator=gen, device="cuda")
    got = ops.token_logprobs(x, tokens, top=top, inv_temperature=inv)
    exactly = torch.tensor(inv, dtype=FP32).double().item()
    logprob, entropy, lse, log_p = _score_exact(x, tokens, exactly)
    # a difference of two logits and its product with 1/T are off by 2^-24 each, the sum of a row by
    # less than 2^-20, and the entropy by that times exponents of a few units that have weight
    for mine, want in ((got.logprob, logprob), (got.entropy, entropy), (got.lse, lse)):
        _agree(mine, want, 2.0 ** -21, 2.0 ** -18)
    if top:
        order = torch.sort(x.float(), dim=1, descending=True, stable=True)[1][:, :top]
        assert torch.equal(got.top_index, order)
        # beyond fp32's range: -inf
        _agree(got.top_logprob, log_p.gather(1, order).float(), 2.0 ** -21, 2.0 ** -18)
