"""The embedding and its gradient against their definition in 64 bits.

Tolerances: the lookup rounds a product once.  A row of the gradient is a
float32 sum of c products in a fixed order, so it is off by at most c + 2 units
2^-24 of the sum of its terms' magnitudes, plus the rounding to 16 bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def op(*a, **k):
    import prlstm_b200 as P

    return P.embedding(*a, **k)


def check(tokens, weight, dout, scale, pad, out, dw):
    tok, dtype = tokens.cpu().long().reshape(-1), weight.dtype
    V, D = weight.shape
    w, d = weight.detach().double().cpu(), dout.double().cpu().reshape(-1, D)
    want = w[tok] * scale
    assert out.dtype == dtype and out.shape == (*tokens.shape, D)
    err = (out.detach().double().cpu().reshape(-1, D) - want).abs()
    assert (err <= (2.0 ** -24 + (UNIT[dtype] if dtype != torch.float32 else 0)) * want.abs() + TINY[dtype]).all()
    keep = tok != pad if pad is not None else torch.ones_like(tok, dtype=torch.bool)
    grad = torch.zeros(V, D, dtype=torch.float64).index_add_(0, tok[keep], d[keep] * scale)
    size = torch.zeros(V, D, dtype=torch.float64).index_add_(0, tok[keep], d[keep].abs() * abs(scale))
    count = torch.bincount(tok[keep], minlength=V)[:, None]
    tol = (count + 2) * 2.0 ** -24 * size + TINY[dtype]
    if dtype != torch.float32:
        tol = tol + UNIT[dtype] * grad.abs()
    err = (dw.double().cpu() - grad).abs()
    assert dw.dtype == dtype and bool((err <= tol).all()), f"off by {float((err - tol).max()):.3e} over"


def run(tokens, V, D, dtype, scale=1.0, pad=None, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    weight = torch.randn(V, D, device=DEV, generator=g).to(dtype).requires_grad_(True)
    dout = torch.randn(*tokens.shape, D, device=DEV, generator=g).to(dtype)
    out = op(tokens, weight, scale=scale, padding_idx=pad)
    out.backward(dout)
    check(tokens, weight, dout, scale, None if pad is None else pad % V, out, weight.grad)
    return out.detach(), weight.grad


def some(n, V, seed, skew=True):
    g = torch.Generator(device=DEV).manual_seed(seed)
    u = torch.rand(n, device=DEV, generator=g)
    return (((V + 1.0) ** u).long().clamp_(1, V) - 1) if skew else (u * V).long().clamp_(max=V - 1)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("N,V,D", [(1, 1, 1), (1, 7, 3), (3, 2, 8), (31, 300, 33), (32, 511, 64), (33, 512, 66), (64, 513, 130),
                                   (1000, 7, 20), (1025, 70000, 12), (4097, 1, 96), (9000, 900, 257), (20011, 262145, 4),
                                   (5000, 40, 1024)])
def test_lookup_and_gradient(N, V, D, dtype):
    run(some(N, V, seed=N + V), V, D, dtype, scale=1.7, seed=D)


@pytest.mark.parametrize("count", [31, 32, 33, 64, 65, 1000, 1055, 1056, 1088, 5000, 40000])
def test_one_token_many_times(count):
    """Runs that end at, before and after the boundaries of the summing pieces,
    alone and between neighbours, up to runs of over a thousand pieces."""
    for before, after in ((0, 0), (1, 1), (31, 40), (32, 0)):
        tok = torch.cat([torch.full((before,), 2), torch.full((count,), 3), torch.full((after,), 5)]).to(DEV)
        tok = tok[torch.randperm(len(tok), device=DEV, generator=torch.Generator(device=DEV).manual_seed(count))]
        run(tok, 6, 36, torch.float32, seed=count)


@pytest.mark.parametrize("kind", [torch.int64, torch.int32])
def test_token_types_shapes_and_strides(kind):
    tok = some(24, 50, 1).to(kind)
    run(tok.view(2, 3, 4), 50, 16, torch.bfloat16)
    run(tok.view(4, 6).t(), 50, 16, torch.bfloat16)  # not contiguous
    run(tok[5], 50, 16, torch.float32)  # a single token without an axis
    run(tok[:0], 50, 16, torch.float32)  # none: an all-zero gradient


def test_padding_row_gets_no_gradient():
    tok = some(3000, 100, 2)
    _, dw = run(tok, 100, 24, torch.float32, pad=0)
    assert not dw[0].any() and dw[1].any()
    _, dw = run(tok, 100, 24, torch.float32, pad=-100)
    assert not dw[0].any()
    _, dw = run(torch.full((70,), 4, device=DEV), 9, 24, torch.float32, pad=4)
    assert not dw.any()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_slices_of_a_table(dtype):
    table = torch.randn(40, 50, device=DEV).to(dtype)
    tok = some(90, 20, 3, skew=False)
    for view in (table[:20, :32], table[20:, 1:34], table[::2, 8:24], table.t()[:20, :16], table[:1].expand(20, 50)):
        leaf = view.detach().requires_grad_(True)
        out = op(tok, leaf, scale=0.5)
        dout = torch.randn(*out.shape, device=DEV).to(dtype)
        out.backward(dout)
        check(tok, leaf, dout, 0.5, None, out, leaf.grad)
    leaf = table[:20, :24].clone().requires_grad_(True)
    op(tok, leaf).sum().backward()  # an expanded gradient
    count = torch.bincount(tok, minlength=20).double()
    assert torch.equal(leaf.grad.double(), count[:, None].expand(20, 24))


def test_ids_out_of_range_are_reported_and_harmless():
    import prlstm_b200 as P

    try:
        w = torch.randn(10, 8, device=DEV, requires_grad=True)
        tok = torch.tensor([3, -1, 10, 2 ** 40, 3, -2 ** 60, 9], device=DEV)
        out = op(tok, w)
        ok = torch.tensor([0, 4, 6], device=DEV)
        assert torch.equal(out[ok], w.detach()[tok[ok]]) and not out[[1, 2, 3, 5]].any()
        out.sum().backward()
        want = torch.zeros(10, 8, device=DEV)
        want[3], want[9] = 2, 1
        assert torch.equal(w.grad, want)
        with pytest.raises(RuntimeError, match="token id"):
            P.check_device_status()
        # the recurrent layers' own waits are not cut short by it
        m = P.HeadStartLSTM(8, 32, parallel=True).to(DEV)
        x = torch.randn(64, 2, 8, device=DEV)
        y = m(x)[0]
        with pytest.raises(RuntimeError, match="token id"):
            op(tok[:1], w)  # reported until it is cleared
    finally:
        P.clear_device_status()
    assert torch.allclose(y, m(x)[0], rtol=1e-5, atol=1e-6)
    P.check_device_status()


def test_same_bits_every_run_and_on_another_stream():
    tok = some(30000, 5000, 4)
    first = run(tok, 5000, 72, torch.float32, seed=1)
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(side):
        again = run(tok, 5000, 72, torch.float32, seed=1)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_long_offsets():
    """A table of more than 2^31 elements, and rows beyond them."""
    V, D = 2_200_000, 1024
    w = torch.empty(V, D, dtype=torch.bfloat16, device=DEV)
    rows = torch.tensor([0, 1_048_576, 2_097_152, 2_199_999], device=DEV)
    w[rows] = torch.randn(4, D, device=DEV).bfloat16()
    assert torch.equal(op(rows, w), w[rows])


def test_refusals():
    w, tok = torch.randn(10, 8, device=DEV), torch.tensor([1, 2], device=DEV)
    for bad, kind in (((tok, w.double()), TypeError), ((tok.float(), w), TypeError), ((tok, w[0]), RuntimeError),
                      ((tok.cpu(), w), RuntimeError), ((tok.cpu(), w.cpu()), RuntimeError)):
        with pytest.raises(kind):
            op(*bad)
    with pytest.raises(RuntimeError):
        op(tok, w, padding_idx=10)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("scale", [1.0, 0.5, -2.0, 20.0 ** 0.5, 0.1, -0.3, 0.0])
def test_infinities_stay(scale, dtype):
    """Rows with infinities and NaN, and gradients of them, are what the product in 64 bits gives."""
    inf, nan = float("inf"), float("nan")
    row = torch.tensor([inf, -inf, nan, 0.0, 1.0, -1.0, 4.0], dtype=torch.float64)
    for D in (7, 8, 300):
        w = row.repeat(D // 7 + 1)[:D].expand(3, D).to(dtype).to(DEV).clone().requires_grad_(True)
        tok = torch.tensor([0, 2, 2, 1], device=DEV)
        dout = row.flip(0).repeat(D // 7 + 1)[:D].expand(4, D).to(dtype).to(DEV)
        out = op(tok, w, scale=scale)
        out.backward(dout)
        want = w.detach().double().cpu()[tok.cpu()] * scale
        grad = torch.stack([dout[0].double().cpu() * n for n in (1, 1, 2)]) * scale
        for got, t in ((out.detach(), want), (w.grad, grad)):
            got = got.double().cpu()
            assert torch.equal(got.isnan(), t.isnan()) and torch.equal(got.isinf(), t.isinf())
            at = t.isinf()
            assert torch.equal(got[at], t[at])
            at = t.isfinite()
            tol = 4 * 2.0 ** -24 + (UNIT[dtype] if dtype != torch.float32 else 0)
            assert ((got[at] - t[at]).abs() <= tol * t[at].abs()).all()
