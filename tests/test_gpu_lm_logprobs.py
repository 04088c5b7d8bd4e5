"""Log probabilities of given tokens, entropy, top alternatives and the
gradient of the logits against their definition in 64 bits.

Tolerances: a base-2 logit t carries two roundings, |t| 2^-23, and enters as
2^t with the hardware exponential's 2^-22; a thread adds up to V / 256 terms in
order.  So log S is off by about (V / 256 + 64) 2^-24 + 2^-21, a log
probability by 2^-22 of its size more, the entropy by the same times the logits'
spread; a gradient by those times its terms, and by its own rounding."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
NINF = -math.inf


def op(*a, **k):
    import prlstm_b200 as P

    return P.token_logprobs(*a, **k)


def truth(logits, tokens, top, T, ignore, g=None, ge=None, gt=None):
    x, tok = logits.detach().double().cpu(), tokens.cpu().long()
    N, V = x.shape
    live = tok != ignore
    empty = (x == NINF).all(1)
    bad = torch.isnan(x).any(1) | (x == math.inf).any(1)
    lp = torch.log_softmax(x / T, 1)
    lp[empty] = NINF
    lp[bad] = math.nan
    p = lp.exp()
    at = tok.clamp(0, V - 1)
    inside = (tok >= 0) & (tok < V)
    pl = torch.where(p > 0, p * lp, torch.where(torch.isnan(p), p, 0.0))
    ent = -pl.sum(1)
    out = dict(logprob=torch.where(live, torch.where(inside, lp.gather(1, at[:, None])[:, 0], math.nan), 0.0),
               entropy=torch.where(live, ent, 0.0))
    if top:
        idx = torch.sort(x + 0.0, dim=1, descending=True, stable=True).indices[:, :top]
        out["top_logprob"] = torch.where(live[:, None], lp.gather(1, idx), 0.0)
        out["top_index"] = torch.where((live & ~bad)[:, None], idx, -1)
    if g is not None or ge is not None or gt is not None:
        zero = torch.zeros(N, dtype=torch.float64)
        g = zero if g is None else torch.where(inside, g.double().cpu(), 0.0)
        ge = zero if ge is None else ge.double().cpu()
        G = g.clone()
        d = torch.zeros(N, V, dtype=torch.float64)
        d.scatter_add_(1, at[:, None], g[:, None])
        if gt is not None:
            d.scatter_add_(1, idx, gt.double().cpu())
            G += gt.double().cpu().sum(1)
        d -= p * G[:, None] + ge[:, None] * (pl + p * ent[:, None])
        d /= T
        d[~live | empty] = 0
        d[bad & live] = math.nan
        out["dlogits"] = d
        p, ent = (torch.where(live[:, None], p, 0.0), torch.where(live, ent, 0.0))
        out["scale"] = (g.abs() + (0 if gt is None else gt.double().cpu().abs().sum(1)) + ge.abs() * (ent + 1)) / T
        out["p"] = p
    return out


def near(got, want, tol, what):
    got, tol = got.double().cpu(), torch.as_tensor(tol).expand(want.shape)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), what
    over = (got - want).abs()[fine] - tol[fine]
    assert not over.numel() or float(over.max()) <= 0, f"{what}: {float(over.max()):.3e} over"


def check(logits, tokens, top=0, T=1.0, ignore=-100, grads=(), seed=0):
    N, V = logits.shape
    rnd = torch.Generator().manual_seed(seed)
    g = torch.randn(N, generator=rnd) if "logprob" in grads else None
    ge = torch.randn(N, generator=rnd) if "entropy" in grads else None
    gt = torch.randn(N, top, generator=rnd) if "top" in grads and top else None
    want = truth(logits, tokens, top, T, ignore, g, ge, gt)
    leaf = logits.detach().requires_grad_(bool(grads))
    r = op(leaf, tokens, top=top, temperature=T, ignore_index=ignore)
    sums = (V / 256 + 64) * 2.0 ** -24 + 2.0 ** -21
    spread = math.log(V) + 2
    assert r.logprob.dtype == r.entropy.dtype == torch.float32
    near(r.logprob.detach(), want["logprob"], sums + 2.0 ** -22 * want["logprob"].abs().nan_to_num(0, 0, 0), "logprob")
    near(r.entropy.detach(), want["entropy"], spread * sums, "entropy")
    if top:
        assert torch.equal(r.top_index.cpu(), want["top_index"]), "top_index"
        near(r.top_logprob.detach(), want["top_logprob"], sums + 2.0 ** -22 * want["top_logprob"].abs().nan_to_num(0, 0, 0), "top_logprob")
    else:
        assert r.top_logprob is None and r.top_index is None
    if grads:
        pairs = [(o, v) for o, v in ((r.logprob, g), (r.entropy, ge), (r.top_logprob, gt)) if v is not None]
        torch.autograd.backward([o for o, _ in pairs], [v.to(DEV) for _, v in pairs])
        d = want["dlogits"]
        # p is off by (|log p| 2^-22 + sums) of itself, and multiplies gradients and, for the entropy's, |log p|
        tol = 4 * sums * spread * (want["scale"][:, None] * want["p"]) + 2.0 ** -22 * want["scale"][:, None] * want["p"].clamp(min=1e-30) * \
            want["p"].clamp(min=1e-30).log().abs() ** 2 + (UNIT[logits.dtype] + 2.0 ** -23) * d.abs() + TINY[logits.dtype]
        named = 2.0 ** -22 * want["scale"][:, None] + torch.zeros_like(d)
        where = torch.zeros_like(d, dtype=torch.bool)
        where.scatter_(1, tokens.cpu().long().clamp(0, V - 1)[:, None], True)
        if gt is not None:
            where.scatter_(1, want["top_index"].clamp(min=0), True)
        near(leaf.grad, d, tol.nan_to_num(0, 0, 0) + torch.where(where, named, 0.0), "dlogits")
        assert leaf.grad.dtype == logits.dtype
    return r


def normal(N, V, dtype, seed, spread=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = (spread * torch.randn(N, V, device=DEV, generator=g)).to(dtype)
    return x, torch.randint(0, V, (N,), device=DEV, generator=g)


SIZES = [(1, 1), (3, 2), (5, 7), (9, 31), (4, 33), (40, 255), (7, 256), (3, 1000), (2, 1024), (5, 1025), (3, 2049), (6, 5000), (2, 50021),
         (1, 131075), (3, 140001), (700, 2200)]
ALL = ("logprob", "entropy", "top")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("N,V", SIZES)
def test_values_and_gradient(N, V, dtype):
    x, tok = normal(N, V, dtype, seed=N + V)
    check(x, tok, grads=("logprob", "entropy"))
    for top in {min(1, V), min(5, V), min(32, V)}:
        check(x, tok, top=top, T=0.7, grads=ALL, seed=top)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_strides_and_alignment(dtype):
    for V, wide, off in ((300, 320, 0), (2201, 2203, 1), (4100, 4115, 3), (9, 64, 5)):
        x, tok = normal(6, wide, dtype, seed=V)
        tok = tok % V
        check(x[:, off:off + V], tok, top=5, grads=ALL)
        check(x[::2, off:off + V], tok[::2], top=5, grads=ALL)
    y = x.t().contiguous().t()  # columns first
    check(y, tok % 64, top=3, grads=ALL)
    x, tok = normal(6, 2200, dtype, seed=1)
    check(x[:1].expand(6, 2200), tok, top=3)


@pytest.mark.parametrize("N,V", [(4, 40), (4, 1000), (3, 5000), (2, 70001), (800, 3000)])
def test_ties_take_the_lowest_index(N, V):
    g = torch.Generator(device=DEV).manual_seed(V)
    tok = torch.randint(0, V, (N,), device=DEV, generator=g)
    few = torch.randint(0, 3, (N, V), device=DEV, generator=g).float()
    for x in (torch.zeros(N, V, device=DEV), few, few.bfloat16(), torch.where(few > 1, 0.0, -0.0)):
        check(x, tok, top=min(32, V), grads=ALL)


@pytest.mark.parametrize("V", [50, 1500, 9000, 70001])
def test_order_of_the_row_does_not_matter(V):
    up = torch.linspace(-4, 4, V, device=DEV)
    block = up.clone()
    block[V // 3: V // 3 + 40] += 20  # the best side by side
    comb = up.clone()
    comb[5::2048] += 20  # the best in one thread's values
    x = torch.stack([up, up.flip(0), block, comb])
    check(x, torch.arange(4, device=DEV), top=32, grads=ALL)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("V", [3, 40, 1500, 6000, 50021])
def test_masks(V, dtype):
    """-inf masks that leave some, one or none; the type's lowest value as a mask."""
    low = torch.finfo(dtype).min
    x, tok = normal(8, V, dtype, seed=V)
    x[0] = NINF
    x[1] = NINF
    x[1, tok[1]] = 1.0
    x[2, : V // 2] = NINF
    x[3, 1:] = low
    x[4] = low
    x[5, ::2] = NINF
    x[6, 0] = NINF  # the token itself is masked out
    tok[6] = 0
    x[7, : V - 1] = NINF
    for top in (0, min(5, V), min(32, V)):
        # gradients of -inf log probabilities (rows 0, 1, 7) name no finite value
        check(x, tok, top=top, grads=("logprob", "entropy"))
        check(x, tok, top=top, T=3.0)


@pytest.mark.parametrize("V", [40, 3000, 70001])
def test_rows_without_a_distribution(V):
    x, tok = normal(6, V, torch.float32, seed=V)
    x[0, V // 2] = math.nan
    x[1, V - 1] = math.inf
    x[2] = math.nan
    x[3, 0] = math.nan
    x[3, 1:] = NINF
    check(x, tok, top=5, grads=("logprob", "entropy"))


def test_large_and_small_logits():
    x, tok = normal(6, 3000, torch.float32, seed=1)
    x[0] += 30000
    x[1] -= 30000
    x[2] *= 1e-3
    x[3, 7] = 3e38
    x[3, 8] = -3e38
    x[4] *= 1e4
    tok[3] = 7
    want = truth(x, tok, 0, 1.0, -100)
    r = op(x, tok)
    near(r.logprob, want["logprob"], 1e-5 + 2.0 ** -22 * want["logprob"].abs(), "logprob")
    near(r.entropy, want["entropy"], torch.tensor(1e-4), "entropy")


def test_ignored_rows_are_not_read():
    x, tok = normal(64, 900, torch.bfloat16, seed=2)
    tok[::3] = -100
    x[::3] = math.nan
    check(x, tok, top=4, grads=ALL)
    tok[:] = -100
    check(x, tok, top=4, grads=("logprob",))
    y, tok = normal(5, 70001, torch.float32, seed=3)
    tok[1:4] = 7
    check(y, tok, top=4, ignore=7, grads=ALL)


def test_tokens_out_of_range_are_reported():
    import prlstm_b200 as P

    for V in (100, 3000, 70001):
        try:
            x, tok = normal(4, V, torch.float32, seed=V)
            tok[1], tok[2] = V, -5
            check(x, tok, top=3, grads=ALL)
            with pytest.raises(RuntimeError, match="token id"):
                P.check_device_status()
        finally:
            P.clear_device_status()
    P.check_device_status()


def test_shapes_types_and_partial_gradients():
    x, tok = normal(24, 50, torch.float32, seed=4)
    flat = op(x, tok, top=3)
    r = op(x.view(2, 3, 4, 50), tok.view(2, 3, 4).int(), top=3)
    assert r.logprob.shape == (2, 3, 4) and r.top_index.shape == (2, 3, 4, 3)
    assert torch.equal(r.logprob.reshape(-1), flat.logprob) and torch.equal(r.top_index.reshape(24, 3), flat.top_index)
    one = op(x[3], tok[3], top=3)
    assert one.logprob.shape == () and torch.equal(one.logprob, flat.logprob[3])
    for grads in (("logprob",), ("entropy",), ("top",), ("logprob", "top")):
        check(x, tok, top=3, grads=grads)
    empty = op(x[:0].requires_grad_(True), tok[:0], top=3)
    assert empty.logprob.shape == (0,) and empty.top_index.shape == (0, 3)
    leaf = x.clone().requires_grad_(True)
    (-op(leaf, tok).logprob.mean()).backward()  # an expanded gradient: cross-entropy
    want = truth(x, tok, 0, 1.0, -100, torch.full((24,), -1 / 24.0))
    near(leaf.grad, want["dlogits"], torch.tensor(1e-7), "cross-entropy")


def test_gradient_against_differences():
    """Central differences, step 2^-4: the third-order term is below 2^-8 / 6 of
    the gradient's scale; results round at about 2^-20 / step."""
    x, tok = normal(3, 11, torch.float32, seed=5, spread=1.0)
    rnd = torch.Generator().manual_seed(6)
    g, ge, gt = torch.randn(3, generator=rnd).to(DEV), torch.randn(3, generator=rnd).to(DEV), torch.randn(3, 2, generator=rnd).to(DEV)

    def loss(x):
        r = op(x, tok, top=2, temperature=1.5)
        return (r.logprob.double() * g).sum() + (r.entropy.double() * ge).sum() + (r.top_logprob.double() * gt).sum()

    leaf = x.clone().requires_grad_(True)
    loss(leaf).backward()
    for i in range(x.numel()):
        up, down = x.clone(), x.clone()
        up.view(-1)[i] += 2.0 ** -4
        down.view(-1)[i] -= 2.0 ** -4
        if not torch.equal(op(up, tok, top=2).top_index, op(down, tok, top=2).top_index):
            continue  # the alternatives change between the two: no derivative to compare
        diff = float(loss(up) - loss(down)) * 2.0 ** 3
        assert abs(diff - float(leaf.grad.view(-1)[i])) <= 2.0 ** -8 * 4, i


def test_same_bits_every_run_and_on_another_stream():
    for N, V in ((2, 131075), (900, 2200)):
        x, tok = normal(N, V, torch.bfloat16, seed=7)
        first = op(x, tok, top=8)
        side = torch.cuda.Stream(DEV)
        side.wait_stream(torch.cuda.current_stream(DEV))
        with torch.cuda.stream(side):
            again = op(x, tok, top=8)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_long_offsets():
    """Logits of more than 2^31 elements."""
    N, V = 33000, 65536
    x = torch.zeros(N, V, dtype=torch.float16, device=DEV)
    tok = torch.full((N,), 9, device=DEV)
    x[N - 1, 5] = 3.0
    r = op(x, tok, top=1)
    assert abs(float(r.logprob[0]) + math.log(V)) < 1e-5
    assert r.top_index[N - 1].tolist() == [5] and abs(float(r.logprob[N - 1]) + math.log(V - 1 + math.exp(3))) < 1e-5


def test_refusals():
    x, tok = normal(4, 20, torch.float32, seed=8)
    with pytest.raises(TypeError):
        op(x.double(), tok)
    with pytest.raises(TypeError):
        op(x, tok.float())
    for args, kw in (((x, tok[:3]), {}), ((x, tok), {"top": 33}), ((x, tok), {"top": 21}), ((x, tok), {"top": -1}),
                     ((x, tok), {"temperature": 0.0}), ((x, tok), {"temperature": float("nan")}), ((x.cpu(), tok.cpu()), {}),
                     ((x, tok.cpu()), {}), ((x[:, :0], tok), {})):
        with pytest.raises(RuntimeError):
            op(*args, **kw)


@pytest.mark.parametrize("default", [torch.float64, torch.bfloat16, torch.float16], ids=str)
def test_results_are_float32_whatever_the_default_dtype(default):
    x = torch.linspace(-3, 3, 5 * 301, dtype=torch.float32, device=DEV).view(5, 301)
    tok = torch.arange(5, device=DEV)

    def run():
        leaf = x.clone().requires_grad_(True)
        r = op(leaf, tok, top=3)
        torch.autograd.backward([r.logprob, r.entropy, r.top_logprob],
                                [torch.ones_like(r.logprob), torch.ones_like(r.entropy), torch.ones_like(r.top_logprob)])
        return [t.detach() for t in r] + [leaf.grad]

    want = run()
    before = torch.get_default_dtype()
    torch.set_default_dtype(default)
    try:
        got = run()
    finally:
        torch.set_default_dtype(before)
    for g, w in zip(got, want):
        assert g.dtype == w.dtype and torch.equal(g, w)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("N,V", [(2, 20000), (600, 20011), (9, 1500), (2048, 3000), (600, 40000)])
def test_alternatives_wherever_they_lie(N, V, dtype):
    """The largest values next to one another, or one thread's vectors, batches or rows' parts apart."""
    strides = [1, 2, 3, 4, 8, 32, 64, 128, 256, 512, 1000, 1024, 2048, 4096, 8192]
    x = torch.zeros(N, V, device=DEV)
    g = torch.Generator().manual_seed(V)
    want = torch.empty(N, 32, dtype=torch.int64)
    for n in range(N):
        stride = strides[n % len(strides)]
        at = (torch.arange(32) * stride + int(torch.randint(V, (1,), generator=g))) % V
        if len(at.unique()) < 32:  # the stride divides the row: wrap to neighbours
            at = torch.arange(32) + n % (V - 32)
        want[n] = at[torch.randperm(32, generator=g)] if n % 3 else at if n % 2 else at.flip(0)
    value = torch.arange(132, 100, -1, dtype=torch.float32, device=DEV)  # exact in every type
    x.scatter_(1, want.to(DEV), value.expand(N, 32))
    for top in (1, 5, 32):
        r = op(x.to(dtype), torch.zeros(N, dtype=torch.int64, device=DEV), top=top)
        assert torch.equal(r.top_index.cpu(), want[:, :top]), top


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("V", [33, 300, 1000])
def test_alternatives_of_many_short_rows(V, dtype):
    """A warp per row, many rows after one another in the same shared memory."""
    N = 20000
    x, tok = normal(N, V, dtype, seed=V)
    for top in (1, 6, 32):
        r = op(x, tok, top=top)
        want = torch.sort(x.double(), dim=1, descending=True, stable=True).indices[:, :top]
        assert torch.equal(r.top_index, want), top
