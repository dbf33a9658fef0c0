"""The decode step's operators at the edges of what their definitions allow, against plain
implementations in 64 bits: temperatures far from one, values at the ends of their types, NaN that
some rows see and others do not, bits lost on the way."""

import math

import pytest
import torch

from newt_b200 import ops
from newt_b200.examples import kernels
from newt_b200.runtime import abi
from test_decode_ops_gpu import (BF16, FP16, FP32, HALF, _attend_exact, _finite_cache, _gen, _int32, _pages, _randn,
                                 _score_exact)

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


@pytest.mark.parametrize("inv", [1e-20, 1e-3, 10.0, 100.0, 1e3, 1e6, 1e9, 1e20])
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("rows, vocab", [(3, 1003), (301, 257)])
def test_token_logprobs_backward_at_far_temperatures(rows, vocab, dtype, inv):
    """No probability above 1, however coarse the row's lse has become."""
    gen = _gen(rows * 5 + vocab)
    x = _randn(gen, rows, vocab, dtype=dtype, scale=3.0)
    x[:, vocab - 7:] = -math.inf
    tokens = torch.randint(0, vocab - 7, (rows,), generator=gen, device="cuda")
    g, ge = _randn(gen, rows), _randn(gen, rows, scale=0.3)
    f = ops.token_logprobs(x, tokens, inv_temperature=inv)
    got = ops.token_logprobs_backward(x, tokens, f.lse, f.entropy, g, ge, inv_temperature=inv).double()
    exactly = torch.tensor(inv, dtype=FP32).double().item()
    _, entropy, lse, log_p = _score_exact(x, tokens, exactly)
    p = log_p.exp()
    hit = torch.zeros_like(p).scatter_(1, tokens[:, None], 1.0)
    inner = torch.where(p > 0, log_p, 0.0) + entropy[:, None]
    want = exactly * (g.double()[:, None] * (hit - p) - ge.double()[:, None] * p * inner)
    # lse and the product of a logit and 1/T are off by 2^-24 of themselves: with d = 2^-21 |lse| more
    # or less in the exponent p lies between p e^-d and min(1, p e^d), and p |log p| up to 1/e + d p
    d = (2.0 ** -21 * lse.abs() + 2.0 ** -18)[:, None]
    high = torch.minimum((log_p + d).exp(), torch.ones_like(p))
    off_p = torch.maximum(high - p, p * -torch.expm1(-d))
    part = ge.abs().double()[:, None] * (high * (d + 2.0 ** -18) + off_p * (inner.abs().clamp(max=1000) + d.clamp(max=1000)))
    # values off by less than a step of a type's smallest normal number may be anything below it
    bound = exactly * (g.abs().double()[:, None] * (off_p + 2.0 ** -22) + part) + HALF[dtype] * want.abs() + exactly * 2.0 ** -20 + 1e-38
    assert torch.isfinite(got).all()
    assert ((got - want).abs() <= bound).all()
    most = exactly * (2 * g.abs() + ge.abs() * (1 + entropy)).double()[:, None] * 1.01
    assert (got.abs() <= most).all()


def test_token_logprobs_backward_of_large_logits():
    """Logits whose lse rounds by several units: no probability comes out above 1."""
    x = torch.full((4, 1000), 1e8, device="cuda")
    x[1] = -1e8
    x[2] = 3e9
    x[3, ::2] = -3e9
    tokens = torch.tensor([3, 4, 5, 6], device="cuda")
    f = ops.token_logprobs(x, tokens, inv_temperature=0.7)
    one = torch.ones(4, device="cuda")
    got = ops.token_logprobs_backward(x, tokens, f.lse, f.entropy, one, inv_temperature=0.7)
    assert got.abs().max() <= 1.0
    got = ops.token_logprobs_backward(x, tokens, f.lse, f.entropy, None, one, inv_temperature=0.7)
    assert got.abs().max() <= 1 + math.log(1000)
    x[0, 0] = math.nan                            # still the row's whole
    f = ops.token_logprobs(x, tokens, inv_temperature=0.7)
    got = ops.token_logprobs_backward(x, tokens, f.lse, f.entropy, one, one, inv_temperature=0.7)
    assert torch.isnan(got[0]).all() and torch.isfinite(got[1:]).all()


def _scores(x, tokens, inv):
    """logprob and entropy in 64 bits, for torch to differentiate."""
    log_p = torch.log_softmax(x * inv, 1)
    p = log_p.exp()
    entropy = -torch.where(p > 0, p * log_p, 0.0).sum(1)
    picked = log_p.gather(1, tokens.clamp(min=0)[:, None])[:, 0]
    return torch.where(tokens < 0, 0.0, picked), entropy


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("top", [0, 4])
def test_token_logprobs_is_differentiated(dtype, top):
    """A training loss through autograd, against the definition differentiated in 64 bits."""
    gen = _gen(95 + top)
    wide = _randn(gen, 33, 1200, dtype=dtype, scale=2.0)
    tokens = torch.randint(0, 1003, (33,), generator=gen, device="cuda")
    tokens[::5] = -100
    weight = _randn(gen, 33)
    losses = {
        "sum": lambda lp, h: -lp.sum() + 0.1 * h.mean(),              # gradients that are broadcast
        "weighted": lambda lp, h: (lp * weight).sum() - (0.01 * h * weight).sum(),
        "logprob": lambda lp, h: lp[::2].mean(), "entropy": lambda lp, h: h.square().sum()}
    for name, loss in losses.items():
        leaf = wide.clone().requires_grad_()
        x = leaf[:, 5:1008]                                           # rows that lie apart, off a boundary
        s = ops.token_logprobs(x, tokens, top=top, inv_temperature=0.8)
        with torch.no_grad():
            plain = ops.token_logprobs(x, tokens, top=top, inv_temperature=0.8)
        assert not plain.logprob.requires_grad
        assert all(a is None and b is None or torch.equal(a, b) for a, b in zip(s, plain))
        loss(s.logprob, s.entropy).backward()
        exactly = wide[:, 5:1008].double().requires_grad_()
        loss(*_scores(exactly, tokens, torch.tensor(0.8).double().item())).backward()
        got, want = leaf.grad[:, 5:1008].double(), exactly.grad
        # one rounding to the logits' type; before it p is off by 2^-19 of itself, times weights of a
        # few units and brackets of up to 2^4, and entropies of up to 7 that are differentiated
        off = (got - want).abs() - (HALF[dtype] * want.abs() + 2.0 ** -14 * want.abs().amax(1, keepdim=True) + 2.0 ** -25)
        assert off.max() <= 0, (name, off.max())
        assert (leaf.grad[:, :5] == 0).all() and (leaf.grad[:, 1008:] == 0).all()


def test_what_token_logprobs_cannot_differentiate_is_refused():
    gen = _gen(96)
    x = _randn(gen, 4, 100).requires_grad_()
    tokens = torch.tensor([1, 2, 3, -1], device="cuda")
    for pick in (lambda s: s.lse, lambda s: s.top_logprob):
        s = ops.token_logprobs(x, tokens, top=3)
        with pytest.raises(NotImplementedError, match="lse and top_logprob"):
            (pick(s).sum() + s.logprob.sum()).backward()
    s = ops.token_logprobs(x, tokens, top=3)
    assert not s.top_index.requires_grad
    grad, = torch.autograd.grad(s.logprob.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()
    y = x * 1.0
    s = ops.token_logprobs(y, tokens)
    ops.token_logprobs_backward(y.detach(), tokens, s.lse.detach(), s.entropy.detach(),
                                torch.ones(4, device="cuda"), out=y.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        s.logprob.sum().backward()
    bare = ops.token_logprobs(x)                       # no tokens: the entropy alone
    assert bare.logprob is None
    bare.entropy.sum().backward()
    assert torch.isfinite(x.grad).all()


def test_writes_count_as_modifications():
    gen = _gen(97)
    x, w = _randn(gen, 4, 64, dtype=BF16), _randn(gen, 64, dtype=BF16)
    out, scales, h = torch.empty_like(x, dtype=ops.E4M3), torch.empty(4, 1, device="cuda"), torch.empty_like(x)
    before = [t._version for t in (out, scales, h, x)]
    ops.rmsnorm(x, w, residual=x, out_dtype=ops.E4M3, out=out, scales=scales, residual_out=h)
    assert [t._version for t in (out, scales, h, x)] == [before[0] + 1, before[1] + 1, before[2] + 1, before[3]]
    cache = ops.new_kv_cache(4, 1, 16, 64)
    before = [t._version for t in cache]
    k = _randn(gen, 3, 1, 64, dtype=BF16)
    ops.kv_append(cache, k, k, _int32([[0]]), _int32([0]), _int32([0, 3]), 3)
    assert [t._version for t in cache] == [n + 1 for n in before]
    q = _randn(gen, 1, 1, 2, 64, dtype=BF16)
    o = torch.empty_like(q)
    version = o._version
    ops.kv_attention(q, cache, _int32([[0]]), _int32([3]), out=o)
    assert o._version == version + 1
    with torch.inference_mode():                       # tensors without a version are written too
        cache = ops.new_kv_cache(4, 1, 16, 64)
    ops.kv_append(cache, k, k, _int32([[0]]), _int32([0]), _int32([0, 3]), 3)
    assert torch.equal(ops.kv_attention(q, cache, _int32([[0]]), _int32([3])), o)


def test_token_logprobs_is_differentiated_in_a_graph_and_on_another_stream():
    gen = _gen(98)
    x = _randn(gen, 40, 5001, dtype=BF16).requires_grad_()
    tokens = torch.randint(0, 5001, (40,), generator=gen, device="cuda")

    def step():
        s = ops.token_logprobs(x, tokens, inv_temperature=1.25)
        return torch.autograd.grad((s.logprob + 0.1 * s.entropy).sum(), x)[0]

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    with torch.no_grad():
        x.copy_(_randn(gen, 40, 5001, dtype=BF16))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, step()) and not torch.equal(got, want)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("vocab", [1003, 50021])
def test_a_row_scores_alike_beside_other_rows(vocab, dtype):
    """The same bits whatever the rows beside it hold, and close ones in calls of other numbers of rows."""
    gen = _gen(vocab)
    row = _randn(gen, 1, vocab, dtype=dtype, scale=3.0)
    one = torch.tensor([17], device="cuda")
    alone = ops.token_logprobs(row, one, top=5)
    for rows in (2, 37, 200, 300, 700):
        results = []
        for _ in range(2):
            x = _randn(gen, rows, vocab, dtype=dtype, scale=3.0)
            x[rows // 2] = row
            got = ops.token_logprobs(x, one.expand(rows).contiguous(), top=5)
            results.append([t[rows // 2] for t in got])
        assert all(torch.equal(a, b) for a, b in zip(*results))
        assert torch.equal(results[0][4], alone.top_index[0])
        for got, want in zip(results[0][:4], alone[:4]):
            # twice the sums' error
            _agree(got, want[0].double(), 2.0 ** -20, 2.0 ** -17)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_rows_that_are_not_finite_score_so(bad):
    """NaN and infinities where the definition has them, whatever path a row takes."""
    gen = _gen(99)
    for rows, vocab in ((3, 1003), (300, 1003), (2, 50021), (160, 33)):
        for dtype in (BF16, FP16, FP32):
            x = _randn(gen, rows, vocab, dtype=dtype)
            x[1, vocab // 3] = bad
            tokens = torch.full((rows,), 3, dtype=torch.int64, device="cuda")
            got = ops.token_logprobs(x, tokens, top=3)
            logprob, entropy, lse, _ = _score_exact(x, tokens, 1.0)
            if bad != -math.inf:
                logprob[1] = entropy[1] = lse[1] = math.nan       # no probability is defined
            for mine, want in ((got.logprob, logprob), (got.entropy, entropy), (got.lse, lse)):
                _agree(mine, want, 2.0 ** -21, 2.0 ** -18)


# ---- rmsnorm -----------------------------------------------------------------------------------

@pytest.mark.parametrize("group", [0, 32, 128])
@pytest.mark.parametrize("n", [64, 257, 4096, 16389])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_rmsnorm_of_weights_at_the_end_of_their_type(dtype, n, group):
    """Outputs above 2^126: the 8-bit numbers are those over the scale, not zeros."""
    gen = _gen(n + group)
    x = 0.5 + torch.rand(5, n, generator=gen, device="cuda")
    x = (x * torch.sign(_randn(gen, 5, n))).to(dtype)
    for size in (2.0 ** 125, 2.0 ** 126, 1.4 * 2.0 ** 126, 2.0 ** 126.9):
        w = torch.full((n,), size, device="cuda").to(dtype)
        got = ops.rmsnorm(x, w, eps=1e-5, out_dtype=ops.E4M3, group=group)
        h = x.double()
        y = h / (h.square().mean(1, keepdim=True) + 1e-5).sqrt() * w.double()
        assert y.abs().max() < torch.finfo(FP32).max
        width = group or n
        scales = torch.stack([part.abs().amax(1) / 448 for part in y.split(width, 1)], 1)
        # the mean's sum, the root and the products: below 2^-17 in all; half a step of e4m3 is 2^-4
        _agree(got.scales, scales, 2.0 ** -17, 0.0)
        q = y / scales.repeat_interleave(width, 1)[:, :n]
        _agree(got.out.float(), q, 2.0 ** -4 + 2.0 ** -15, 2.0 ** -10 * 1.001)


def test_rmsnorm_of_rows_without_columns():
    x, w = torch.zeros(3, 0, device="cuda", dtype=BF16), torch.zeros(0, device="cuda", dtype=BF16)
    scales = torch.full((3, 1), 7.0, device="cuda")
    got = ops.rmsnorm(x, w, out_dtype=ops.E4M3, scales=scales)
    assert got.out.shape == (3, 0) and (scales == 1).all()          # the scale of nothing
    assert ops.rmsnorm(x, w, out_dtype=ops.E4M3, group=32).scales.shape == (3, 0)
    assert ops.rmsnorm(x, w).out.shape == (3, 0)


@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("rows, n", [(1, 1), (3, 64), (700, 100), (5, 1003), (700, 1003), (2, 4096), (300, 8192),
                                     (2, 32768), (2, 32761)])
def test_rmsnorm_of_rows_whose_squares_leave_the_range(rows, n, dtype, with_residual):
    """Values whose squares are infinite or 0 in fp32, beside ordinary rows of the same call."""
    gen = _gen(rows + n)
    sizes = [1.0, 1e18, 3e19, 1e30, 1e37, 1e-18, 1e-22, 1e-30, 1e-36, 1.0]
    x = _randn(gen, rows, n).clamp(-3, 3)
    x = (x * torch.tensor([sizes[(i + n) % len(sizes)] for i in range(rows)], device="cuda")[:, None]).to(dtype)
    residual = (x * _randn(gen, rows, 1).clamp(-3, 3)).to(dtype) if with_residual else None
    w = _randn(gen, n, dtype=dtype)
    for eps in (0.0, 1e-40, 1e-12, 1e-6):
        eps = torch.tensor(eps, dtype=FP32).item()
        h = x.double() + (residual.double() if with_residual else 0.0)
        want = h / (h.square().mean(1, keepdim=True) + eps).sqrt() * w.double()
        got = ops.rmsnorm(x, w, residual=residual, eps=eps)
        # fp32's own sum of x and the residual: 2^-24 of the larger, relative to the row's size
        slack = 2.0 ** -23 * want.abs().amax(1, keepdim=True) if with_residual else 0.0
        off = (got.out.double() - want).abs() - ((HALF[dtype] + 2.0 ** -17) * want.abs() + 4 * slack + 1e-38)
        assert off.max() <= 0, (eps, off.max())
        if with_residual:
            _agree(got.residual, h, HALF[dtype] + 2.0 ** -23, 1e-38)
        got = ops.rmsnorm(x, w, residual=residual, eps=eps, out_dtype=ops.E4M3, group=32)
        scales = torch.stack([part.abs().amax(1) / 448 for part in want.split(32, 1)], 1)
        usual = scales > 1.2e-38
        assert ((got.scales.double() - scales).abs()[usual] <= (2.0 ** -16 * scales + (slack if with_residual else 0.0))[usual]).all()


@pytest.mark.parametrize("rows, n", [(3, 64), (700, 1003), (5, 4096)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_rmsnorm_of_rows_that_are_not_finite(bad, rows, n):
    """NaN and infinities where the formula has them: every output of a row with NaN, and where a row's
    infinity is; its other outputs are 0."""
    gen = _gen(rows + n)
    for dtype in (BF16, FP16, FP32):
        x, w = _randn(gen, rows, n, dtype=dtype), _randn(gen, n, dtype=dtype)
        x[1, n // 2] = bad
        h = x.double()
        want = h / (h.square().mean(1, keepdim=True) + 1e-6).sqrt() * w.double()
        got = ops.rmsnorm(x, w)
        _agree(got.out, want, HALF[dtype] + 2.0 ** -17, 2.0 ** -24)
        got = ops.rmsnorm(x, w, residual=torch.zeros_like(x))
        _agree(got.residual, h, 0.0, 0.0)
        for group in (0, 32):
            got = ops.rmsnorm(x, w, out_dtype=ops.E4M3, group=group)
            keep = torch.ones(rows, dtype=torch.bool, device="cuda")
            keep[1] = False
            assert torch.isfinite(got.out.float()[keep]).all() and torch.isfinite(got.scales[keep]).all()
            nan = torch.isnan(got.out.float()[1])
            assert nan.all() if math.isnan(bad) else nan.nonzero().tolist() == [[n // 2]]


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_rmsnorm_agrees_with_the_generated_kernel(dtype):
    """The same norm through the block language: fp32 sums on both sides, one rounding each."""
    gen = _gen(12)
    for rows, n in ((7, 64), (300, 1000), (64, 4096)):
        x, w = _randn(gen, rows, n, dtype=dtype), _randn(gen, n, dtype=dtype)
        mine, other = ops.rmsnorm(x, w, eps=1e-5).out, kernels.rmsnorm(x, w, eps=1e-5)
        _agree(mine, other, 2 * HALF[dtype] + 2.0 ** -16, 2.0 ** -24)


# ---- attention over the cache ------------------------------------------------------------------

def _check_some_nan(got, q, cache, table, lengths, window, sinks):
    """NaN where the definition has NaN and nowhere else; the others as close as they have to be."""
    want, _ = _attend_exact(q, cache, table, lengths, q.shape[3] ** -0.5, window, sinks)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    nan = torch.isnan(want)
    clean = cache._replace(**{name: torch.where(torch.isnan(t.float()), 0, t.view(torch.uint8)).view(ops.E4M3)
                              for name, t in (("k", cache.k), ("v", cache.v))})
    assert nan.any() and not nan.all()
    # the same values without NaN: what does not depend on them agrees
    other, size = _attend_exact(q, clean, table, lengths, q.shape[3] ** -0.5, window, sinks)
    assert torch.equal(other[~nan], want[~nan])
    extra = {BF16: 2.0 ** -9 + 2.0 ** -11, FP16: 2.0 ** -11}[q.dtype] + 2.0 ** -11 + 2.0 ** -14
    off = (got.double() - other).abs() - (HALF[q.dtype] * other.abs() + extra * size + 2.0 ** -25)
    assert off[~nan].max() <= 0


@pytest.mark.parametrize("window, sinks", [(0, 0), (40, 3), (5, 0), (300, 1)])
@pytest.mark.parametrize("page, d, heads, kv_heads, nq, dtype", [
    (16, 64, 2, 2, 4, FP16), (16, 128, 4, 2, 2, BF16), (64, 128, 7, 1, 3, BF16), (32, 64, 8, 1, 5, FP16),
    (128, 128, 8, 2, 8, FP16), (64, 64, 3, 3, 4, BF16)])
def test_attention_keeps_nan_from_queries_that_do_not_see_it(page, d, heads, kv_heads, nq, dtype, window, sinks):
    """Value rows with NaN in some columns, seen by some of the call's queries: behind the others' own
    position, or before their window.  Sequences shorter than the queries among them."""
    gen = _gen(page + d + nq + window)
    lengths = [nq + 1, max(nq - 1, 1), 129, 257, 300, 777, 64]
    table, total = _pages(gen, lengths, page)
    cache = _finite_cache(gen, total, kv_heads, page, d)
    for b, n in enumerate(lengths):
        tokens = [n - 1, n - 2] if b % 2 else [n - 1]
        if window and n > nq + window:
            tokens.append(n - nq - window + 1)             # the first query's oldest
        for t in tokens:
            codes = cache.v.view(torch.uint8)[table[b, t // page].item(), b % kv_heads, t % page]
            codes[torch.tensor([3, 17, d - 1, 32 + b], device="cuda")] = torch.tensor(
                [0x7F, 0xFF, 0x7F, 0xFF], dtype=torch.uint8, device="cuda")
    q = _randn(gen, len(lengths), nq, heads, d, dtype=dtype)
    lengths = _int32(lengths)
    got = ops.kv_attention(q, cache, table, lengths, window=window, sinks=sinks)
    _check_some_nan(got, q, cache, table, lengths, window, sinks)
    cache.k.view(torch.uint8)[table[4, (lengths[4].item() - 1) // page].item(), 0, (lengths[4].item() - 1) % page, 5] = 0x7F
    got = ops.kv_attention(q, cache, table, lengths, window=window, sinks=sinks)
    _check_some_nan(got, q, cache, table, lengths, window, sinks)
    for _ in range(2):                                     # and again: nothing of it stays
        again = ops.kv_attention(q, cache, table, lengths, window=window, sinks=sinks)
        assert torch.equal(again.view(torch.int16), got.view(torch.int16))


def test_attention_keeps_nan_from_one_item_to_the_next():
    """Many short items one after another in a share, every third with NaN in its last value row."""
    gen = _gen(77)
    lengths = [5 + (i * 13) % 200 for i in range(300)]
    table, total = _pages(gen, lengths, 16)
    cache = _finite_cache(gen, total, 3, 16, 64)
    for b in range(0, 300, 3):
        t = lengths[b] - 1
        cache.v.view(torch.uint8)[table[b, t // 16].item(), b % 2, t % 16, b % 64] = 0x7F
    q = _randn(gen, 300, 2, 6, 64, dtype=BF16)
    lengths = _int32(lengths)
    got = ops.kv_attention(q, cache, table, lengths)
    _check_some_nan(got, q, cache, table, lengths, 0, 0)


@pytest.mark.parametrize("group, nq, dtype", [(16, 20, FP16), (8, 20, BF16), (16, 9, BF16), (5, 33, FP16)])
def test_attention_keeps_nan_within_its_item_while_the_next_ones_are_staged(group, nq, dtype):
    """Items of one tile each, whose rows see the NaN of their sequence or see nothing, one after another:
    some warps are two items further while others still look at the tile."""
    gen = _gen(group + nq)
    lengths = [1 + (i * 7) % (nq + 3) for i in range(60)]
    table, total = _pages(gen, lengths, 16)
    for d in (64, 128):
        cache = _finite_cache(gen, total, 1, 16, d)
        for b, n in enumerate(lengths):
            for t in range(b % 2, n, 2):
                codes = cache.v.view(torch.uint8)[table[b, t // 16].item(), 0, t % 16]
                codes[torch.randint(0, d, (3,), generator=gen, device="cuda")] = 0x7F
        q = _randn(gen, 60, nq, group, d, dtype=dtype)
        at = _int32(lengths)
        calls = [ops.kv_attention(q, cache, table, at) for _ in range(20)]
        _check_some_nan(calls[0], q, cache, table, at, 0, 0)
        for got in calls[1:]:
            assert torch.equal(got.view(torch.int16), calls[0].view(torch.int16))


def test_attention_of_more_rows_than_a_tile_keeps_nan_where_it_is_seen():
    """Row tiles of 16 rows, some of which none of a token's queries is in; parts of cut items."""
    gen = _gen(78)
    lengths = [3000, 41]
    table, total = _pages(gen, lengths, 32)
    cache = _finite_cache(gen, total, 1, 32, 128)
    for b, t in ((0, 2990), (0, 2999), (0, 1000), (1, 33)):
        cache.v.view(torch.uint8)[table[b, t // 32].item(), 0, t % 32, 7 + t % 100] = 0xFF
    q = _randn(gen, 2, 20, 4, 128, dtype=BF16)
    lengths = _int32(lengths)
    for window, sinks in ((0, 0), (30, 2), (1995, 0)):
        got = ops.kv_attention(q, cache, table, lengths, window=window, sinks=sinks)
        _check_some_nan(got, q, cache, table, lengths, window, sinks)


@pytest.mark.parametrize("d, heads, nq", [(64, 4, 1), (128, 8, 1), (64, 8, 2)])
def test_attention_weighs_fp16_queries_to_14_bits(d, heads, nq):
    """Values of both signs that nearly cancel, so that the output's own rounding is small and what is
    left are the probabilities' bits."""
    gen = _gen(d + heads)
    lengths = [2, 3, 4, 5, 6, 8, 10, 17] * 8
    table, total = _pages(gen, lengths, 16)
    cache = _finite_cache(gen, total, 1, 16, d)
    v = cache.v.view(torch.uint8)
    v[:, :, 1::2] = v[:, :, 0::2] ^ 0x80
    q = _randn(gen, len(lengths), nq, heads, d, dtype=FP16, scale=0.05)
    lengths = _int32(lengths)
    got = ops.kv_attention(q, cache, table, lengths)
    want, size = _attend_exact(q, cache, table, lengths, d ** -0.5, 0, 0)
    # three e4m3 parts: the first leaves up to half its step, 2^-4, the second up to half the step of
    # a number below 2^-4, 2^-9, the third 2^-14, of a probability in [1, 2); scores of a few units in
    # fp32 and their exponentials are below 2^-16
    off = (got.double() - want).abs() - (HALF[FP16] * want.abs() + (2.0 ** -14 + 2.0 ** -16) * size + 2.0 ** -25)
    assert off.max() <= 0, off.max()


@pytest.mark.parametrize("dtype, parts", [(BF16, 2), (FP16, 3)])
def test_attention_of_queries_far_apart_in_size(dtype, parts):
    """Elements far below their row's largest enter with the bits that e4m3's smallest steps leave them."""
    gen = _gen(83)
    table, total = _pages(gen, [90, 300], 32)
    cache = _finite_cache(gen, total, 1, 32, 64)
    lengths = _int32([90, 300])
    for low in range(10, 25, 2):
        q = _randn(gen, 2, 1, 4, 64, dtype=FP32) * 2.0 ** -low
        q[..., 5] = 1.0
        q = (q * 8).to(dtype)
        cache.k.view(torch.uint8)[..., 5] = 0                     # the largest element meets nothing
        got = ops.kv_attention(q, cache, table, lengths, scale=2.0 ** low / 64)
        want, size = _attend_exact(q, cache, table, lengths, 2.0 ** low / 64, 0, 0)
        # half a step of the last part: 2^-10 16^-(parts - 1) where the row's largest is at least 224; so
        # much of 8 / 224 per element, times the keys' magnitudes (below 2^5 2^-5) and the scale: what a
        # score may be off by, and with it a probability's logarithm
        score = 2.0 ** -10 * 16.0 ** (1 - parts) * 8 / 224 * 64 * 2.0 ** low / 64
        extra = {2: 2.0 ** -9, 3: 2.0 ** -11}[parts] + 2.0 ** -11 + 2.0 ** -14 + math.expm1(2 * score)
        off = (got.double() - want).abs() - (HALF[dtype] * want.abs() + extra * size + 2.0 ** -25)
        assert off.max() <= 0, (low, off.max())
