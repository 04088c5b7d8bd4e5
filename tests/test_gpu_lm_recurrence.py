"""The gated linear recurrence against its definition, step by step in 64 bits.

Tolerances, from the float32 arithmetic: a gate carries a relative error of a
few units 2^-24, and an error made in one step lasts as long as the state's
memory, 1 / (1 - |f|) steps at most.  So a state, or a gradient, is off by at
most about 8 units x (memory + 4) of the tensor's largest value, and results
stored in 16 bits by half a unit in their last place more."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(T, B, H, dtype, form, seed=0, starts=False):
    g = torch.Generator().manual_seed(seed)
    if form == "gated":
        a = (1.5 * torch.randn(T, B, H, generator=g) + 1.0).clamp(-6, 5)
    else:
        a = 1.9 * torch.rand(T, B, H, generator=g) - 0.95
    b = torch.randn(T, B, H, generator=g)
    h0 = torch.randn(B, H, generator=g)
    dh, dh_n = torch.randn(T, B, H, generator=g), torch.randn(B, H, generator=g)
    s = torch.rand(T, B, generator=g) < 0.05 if starts else None
    return a.to(dtype), b.to(dtype), h0, s, dh.to(dtype), dh_n


def truth(a, b, h0, s, dh, dh_n, form):
    """h, h_n and the gradients in 64 bits, by the definition, and the memory."""
    a, x, h0 = a.double().cpu(), b.double().cpu(), h0.double().cpu()
    T = a.shape[0]
    f = torch.sigmoid(a) if form == "gated" else a
    om = torch.sigmoid(-a) if form == "gated" else None
    keep = f.clone()
    cut = torch.zeros(a.shape[:2], dtype=torch.bool) if s is None else s.cpu()
    keep[cut] = 0
    inp = om * x if form == "gated" else x
    h, before, state = torch.empty_like(a), torch.empty_like(a), h0
    for t in range(T):
        before[t] = torch.where(cut[t][:, None], 0.0, state)
        state = torch.where(cut[t][:, None], 0.0, f[t] * state) + inp[t]
        h[t] = state
    u = torch.zeros_like(h0) if dh_n is None else dh_n.double().cpu()
    da, db = torch.empty_like(a), torch.empty_like(a)
    for t in range(T - 1, -1, -1):
        e = u + (0 if dh is None else dh[t].double().cpu())
        da[t] = e * (before[t] - x[t]) * f[t] * om[t] if form == "gated" else e * before[t]
        db[t] = e * om[t] if form == "gated" else e
        u = keep[t] * e
    memory = float(1 / (1 - f.abs().max())) if T else 1.0
    return dict(h=h, h_n=state, da=da, db=db, dh0=u), min(memory, T)


def check(got, want, memory, what, dtype=None):
    dtype = dtype or got.dtype
    assert got.dtype == dtype and got.shape == want.shape, what
    if not want.numel():
        return
    err = (got.double().cpu() - want).abs()
    tol = 8 * 2.0 ** -24 * (memory + 4) * want.abs().max() + TINY[dtype]
    if dtype != torch.float32:
        tol = tol + UNIT[dtype] * want.abs()
    worst = float((err - tol).max())
    assert worst <= 0, f"{what}: off by {float(err.max()):.3e}, {worst:.3e} over"


def call(form):
    import prlstm_b200 as P

    return P.gated_recurrence if form == "gated" else P.linear_recurrence


def run(a, b, h0, s, dh, dh_n, form, batch_first=False):
    leaves = [t.to(DEV).requires_grad_(True) if t is not None else None for t in (a, b, h0)]
    h, h_n = call(form)(*leaves[:2], leaves[2], starts=None if s is None else s.to(DEV), batch_first=batch_first)
    outs = [(o, g.to(DEV)) for o, g in ((h, dh), (h_n, dh_n)) if g is not None]
    torch.autograd.backward([o for o, _ in outs], [g for _, g in outs])
    return dict(h=h.detach(), h_n=h_n.detach(), da=leaves[0].grad, db=leaves[1].grad,
                dh0=None if h0 is None else leaves[2].grad)


def check_all(got, want, memory, what):
    for k in ("h", "h_n", "da", "db", "dh0"):
        if got[k] is not None:
            check(got[k], want[k], memory, f"{what} {k}")


SHAPES = [(1, 1, 1), (1, 3, 5), (2, 1, 33), (15, 2, 64), (16, 2, 64), (17, 3, 31), (33, 1, 34), (129, 1, 96),
          (300, 4, 7), (1000, 2, 130), (2049, 1, 64), (5000, 1, 32), (64, 40, 256)]


@pytest.mark.parametrize("form", ["gated", "linear"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward_and_gradient(shape, dtype, form):
    for starts in (False, True):
        a, b, h0, s, dh, dh_n = make(*shape, dtype, form, seed=sum(shape), starts=starts)
        want, memory = truth(a, b, h0, s, dh, dh_n, form)
        check_all(run(a, b, h0, s, dh, dh_n, form), want, memory, f"{shape} starts={starts}")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_batch_first_is_the_transpose(dtype):
    a, b, h0, s, dh, dh_n = make(77, 3, 40, dtype, "gated", seed=3, starts=True)
    want, memory = truth(a, b, h0, s, dh, dh_n, "gated")
    t = lambda x: x.transpose(0, 1).contiguous()  # noqa: E731
    got = run(t(a), t(b), h0, t(s), t(dh), dh_n, "gated", batch_first=True)
    for k in ("h", "da", "db"):
        assert got[k].is_contiguous()
        got[k] = got[k].transpose(0, 1)
    check_all(got, want, memory, "batch first")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_slices_and_odd_alignment_are_read_in_place(dtype):
    """z and x as the halves of one projection, as every second sequence, and
    one element off alignment; gradients of an expanded tensor."""
    T, B, H = 40, 6, 24
    a, b, h0, s, dh, dh_n = make(T, B, H, dtype, "gated", seed=5)
    want, memory = truth(a, b, h0, None, dh, dh_n, "gated")
    both = torch.cat((a, b), 2).to(DEV)
    z, x = both.chunk(2, 2)
    assert not z.is_contiguous()
    h, h_n = call("gated")(z, x, h0.to(DEV))
    check(h, want["h"], memory, "halves")
    wide = torch.zeros(T, 2 * B, H, dtype=dtype, device=DEV)
    wide[:, ::2] = a.to(DEV)
    h, _ = call("gated")(wide[:, ::2], x, h0.to(DEV))
    check(h, want["h"], memory, "every second sequence")
    off = torch.zeros(T * B * H + 1, dtype=dtype, device=DEV)[1:].view(T, B, H)
    off.copy_(a)
    z = off.requires_grad_(True)
    h, h_n = call("gated")(z, x, h0.to(DEV))
    torch.autograd.backward((h, h_n), (dh.to(DEV), dh_n.to(DEV)))
    check(h.detach(), want["h"], memory, "odd alignment")
    check(z.grad, want["da"], memory, "odd alignment da")
    ones, _ = truth(a, b, h0, None, torch.ones_like(dh), None, "gated")
    z2, x2 = a.to(DEV).requires_grad_(True), b.to(DEV).requires_grad_(True)
    call("gated")(z2, x2, h0.to(DEV))[0].sum().backward()  # an expanded gradient
    check(z2.grad, ones["da"], memory, "expanded da")
    check(x2.grad, ones["db"], memory, "expanded db")


@pytest.mark.parametrize("form", ["gated", "linear"])
def test_optional_inputs_and_gradients(form):
    a, b, h0, s, dh, dh_n = make(50, 2, 36, torch.float32, form, seed=7)
    zero = torch.zeros_like(h0)
    for d, dn, start in ((dh, None, None), (None, dh_n, h0), (dh, dh_n, h0.bfloat16())):
        want, memory = truth(a, b, zero if start is None else start, None, d, dn, form)
        got = run(a, b, start, None, d, dn, form)
        if start is not None and start.dtype != torch.float32:
            assert got["dh0"].dtype == start.dtype
            check(got["dh0"], want["dh0"], memory, "dh0 in its own type", start.dtype)
            got["dh0"] = None
        check_all(got, want, memory, f"{form} {d is None} {dn is None}")


def test_broadcast_inputs_and_a_second_backward():
    """Gates shared by all sequences and a state shared by all columns come in
    as expanded tensors; their gradients are the sums.  The graph can be walked twice."""
    T, B, H = 37, 4, 48
    a, b, h0, s, dh, dh_n = make(T, B, H, torch.float32, "gated", seed=23)
    a, h0 = a[:, :1], h0[:, :1]
    want, memory = truth(a.expand(T, B, H), b, h0.expand(B, H), None, dh, dh_n, "gated")
    z, x, start = (t.to(DEV).requires_grad_(True) for t in (a, b, h0))
    h, h_n = call("gated")(z.expand(T, B, H), x, start.expand(B, H))
    check(h.detach(), want["h"], memory, "h")
    for n in (1, 2):
        torch.autograd.backward((h, h_n), (dh.to(DEV), dh_n.to(DEV)), retain_graph=True)
        check(z.grad / n, want["da"].sum(1, keepdim=True), 2 * memory, "da")
        check(x.grad / n, want["db"], memory, "db")
        check(start.grad / n, want["dh0"].sum(1, keepdim=True), 2 * memory, "dh0")


def test_empty_extents():
    for T, B, H in ((0, 3, 8), (4, 0, 8), (4, 3, 0), (0, 0, 0)):
        z = torch.randn(T, B, H, device=DEV, requires_grad=True)
        x = torch.randn(T, B, H, device=DEV, requires_grad=True)
        h0 = torch.randn(B, H, device=DEV, requires_grad=True)
        h, h_n = call("gated")(z, x, h0)
        assert h.shape == (T, B, H) and h_n.shape == (B, H)
        if T == 0:
            assert torch.equal(h_n, h0)
        (h.sum() + 3 * h_n.sum()).backward()
        assert z.grad.shape == z.shape
        if T == 0:
            assert torch.equal(h0.grad, torch.full_like(h0, 3))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_nothing_passes_a_start(dtype):
    """NaN and infinities in one document leave the next one untouched, in
    both directions, wherever the boundary lies among tiles."""
    for T, at in ((40, 7), (40, 16), (700, 513), (3000, 1600)):
        a, b, h0, s, dh, dh_n = make(T, 2, 64, dtype, "gated", seed=at)
        s = torch.zeros(T, 2, dtype=torch.bool)
        s[at] = True
        clean, memory = truth(a, b, h0, s, dh, dh_n, "gated")
        for bad in (float("nan"), float("inf"), -float("inf")):
            bb, hh = b.clone(), h0.clone()
            bb[:at] = bad
            hh[:] = bad
            got = run(a, bb, hh, s, dh, dh_n, "gated")
            check(got["h"][at:], clean["h"][at:], memory, f"h after {bad}")
            check(got["da"][at:], clean["da"][at:], memory, f"da after {bad}")
            check(got["db"], clean["db"], memory, f"db with {bad}")  # does not depend on x
            d = dh.clone()
            d[at:] = bad
            got = run(a, b, h0, s, d, dh_n, "gated")
            check(got["da"][:at], clean["da"][:at], memory, f"da before {bad}")
            check(got["db"][:at], clean["db"][:at], memory, f"db before {bad}")


def test_nan_spreads_as_step_by_step():
    """Without a start a NaN reaches every later state of its column only."""
    a, b, h0, s, dh, dh_n = make(900, 1, 70, torch.float32, "gated", seed=9)
    b[300, 0, 5] = float("nan")
    h, h_n = call("gated")(a.to(DEV), b.to(DEV), h0.to(DEV))
    bad = torch.isnan(h).cpu()
    assert bad[300:, 0, 5].all() and not bad[:300].any() and int(bad.sum()) == 600
    assert torch.isnan(h_n[0, 5])


def test_extreme_gates_and_zero_states():
    T, H = 2100, 32
    z = torch.full((T, 1, H), 200.0, device=DEV)  # f = 1: the state is carried unchanged
    x = torch.randn(T, 1, H, device=DEV)
    h0 = torch.randn(1, H, device=DEV)
    h, h_n = call("gated")(z, x, h0)
    assert torch.equal(h_n, h0) and torch.equal(h, h0.expand(T, 1, H))
    h, h_n = call("gated")(-z, x, h0)  # f = 0: the input passes
    assert torch.equal(h, x)
    # from a zero state, coefficients above 1 whose product overflows give 0
    h, h_n = call("linear")(torch.full((T, 1, H), 2.0, device=DEV), torch.zeros(T, 1, H, device=DEV))
    assert torch.equal(h, torch.zeros_like(h)) and torch.equal(h_n, torch.zeros_like(h_n))


@pytest.mark.parametrize("form", ["gated", "linear"])
def test_gradient_against_differences(form):
    """Central differences of the float32 results: with a step of 2^-5 the
    third-order term is about 2^-10 / 6 of the gradient's scale and the
    rounding of the loss (summed in 64 bits) far below it."""
    a, b, h0, s, dh, dh_n = make(35, 2, 6, torch.float32, form, seed=11, starts=True)
    got = run(a, b, h0, s, dh, dh_n, form)
    step = 2.0 ** -5

    def loss(a, b, h0):
        h, h_n = call(form)(a.to(DEV), b.to(DEV), h0.to(DEV), starts=s.to(DEV))
        return float((h.double().cpu() * dh).sum() + (h_n.double().cpu() * dh_n).sum())

    g = torch.Generator().manual_seed(1)
    for name, k in (("da", 0), ("db", 1), ("dh0", 2)):
        flat = got[name].cpu().reshape(-1)
        for i in torch.randint(0, flat.numel(), (12,), generator=g).tolist():
            d = []
            for sign in (1, -1):
                v = [a.clone(), b.clone(), h0.clone()]
                v[k].view(-1)[i] += sign * step
                d.append(loss(*v))
            diff = (d[0] - d[1]) / (2 * step)
            assert abs(diff - float(flat[i])) <= 2.0 ** -9 * float(flat.abs().max()), (name, i)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_step_equals_the_recurrence(dtype):
    import prlstm_b200 as P

    a, b, h0, _, _, _ = make(6, 5, 70, dtype, "gated", seed=13)
    h, h_n = P.gated_recurrence(a.to(DEV), b.to(DEV), h0.to(DEV))
    state, fresh = h0.to(DEV).clone(), h0.to(DEV)
    for t in range(6):
        o, new = P.gated_recurrence_step(a[t].to(DEV), b[t].to(DEV), fresh)
        out, same = P.gated_recurrence_step(a[t].to(DEV), b[t].to(DEV), state, out_state=state)
        assert same.data_ptr() == state.data_ptr() and torch.equal(state, new) and torch.equal(o, out)
        fresh = new
        want, memory = truth(a[:t + 1], b[:t + 1], h0, None, None, None, "gated")
        check(o, want["h"][t], memory, "step")
    check(state, want["h_n"], memory, "state")
    check(h_n, want["h_n"], memory, "h_n")


def test_second_derivatives_are_refused():
    z = torch.randn(5, 2, 8, device=DEV, requires_grad=True)
    x = torch.randn(5, 2, 8, device=DEV, requires_grad=True)
    h, _ = call("gated")(z, x)
    (g,) = torch.autograd.grad(h.square().sum(), z, create_graph=True)  # the first may be asked for with a graph
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


def test_same_bits_every_run_and_on_another_stream():
    a, b, h0, s, dh, dh_n = make(1500, 2, 200, torch.bfloat16, "gated", seed=17, starts=True)
    first = run(a, b, h0, s, dh, dh_n, "gated")
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(side):
        again = run(a, b, h0, s, dh, dh_n, "gated")
    side.synchronize()
    for k in first:
        assert torch.equal(first[k], again[k]), k


def test_long_offsets():
    """A tensor whose offsets pass 2^31 elements, read through a slice."""
    T, B, H, W = 3, 2, 64, 600_000_000
    big = torch.empty(5 * W + H, dtype=torch.bfloat16, device=DEV).as_strided((T, B, H), (2 * W, W, 1))
    a, b, h0, _, _, _ = make(T, B, H, torch.bfloat16, "gated", seed=19)
    big.copy_(a)
    want, memory = truth(a, b, h0, None, None, None, "gated")
    h, _ = call("gated")(big, b.to(DEV), h0.to(DEV))
    check(h, want["h"], memory, "long offsets")


def test_refusals():
    import prlstm_b200 as P

    z = torch.randn(4, 2, 8, device=DEV)
    with pytest.raises(TypeError):
        P.gated_recurrence(z.double(), z.double())
    with pytest.raises(TypeError):
        P.gated_recurrence(z, z.bfloat16())
    with pytest.raises(RuntimeError):
        P.gated_recurrence(z, z[:, :1])
    with pytest.raises(RuntimeError):
        P.gated_recurrence(z[0], z[0])
    with pytest.raises(RuntimeError):
        P.gated_recurrence(z, z, torch.zeros(3, 8, device=DEV))
    with pytest.raises(RuntimeError):
        P.gated_recurrence(z, z, starts=torch.zeros(2, 4, dtype=torch.bool, device=DEV))
    with pytest.raises(RuntimeError):
        P.gated_recurrence(z, z, starts=torch.zeros(4, 2, device=DEV))
    with pytest.raises(RuntimeError):
        P.gated_recurrence(z.cpu(), z.cpu())
    with pytest.raises(RuntimeError):
        P.gated_recurrence(z, z, torch.zeros(2, 8))
    with pytest.raises(TypeError):
        P.gated_recurrence_step(z[0], z[0], torch.zeros(2, 8, device=DEV, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError):
        P.gated_recurrence_step(z[0], z[0], torch.zeros(2, 8, device=DEV), out_state=torch.zeros(2, 16, device=DEV)[:, ::2])
    with pytest.raises(RuntimeError):
        P.gated_recurrence_step(z[0].requires_grad_(True), z[0], torch.zeros(2, 8, device=DEV))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("T,B,H", [(33, 1, 2), (100, 1, 6), (200, 1, 70), (97, 3, 94), (530, 1, 258), (70, 150, 46)])
def test_rows_off_16_bytes(T, B, H, dtype):
    """Rows that are 4-byte but not 16-byte aligned, alone and as slices, down
    to rows shorter than a granule and up to the tensor's very last bytes."""
    a, b, h0, s, dh, dh_n = make(T, B, H, dtype, "gated", seed=T + H, starts=True)
    for starts in (None, s):
        want, memory = truth(a, b, h0, starts, dh, dh_n, "gated")
        check_all(run(a, b, h0, starts, dh, dh_n, "gated"), want, memory, f"starts={starts is not None}")
    both = torch.cat((a, b), 2).to(DEV).requires_grad_(True)  # halves of one tensor
    z, x = both.chunk(2, 2)
    want, memory = truth(a, b, h0, None, dh, dh_n, "gated")
    h, h_n = call("gated")(z, x, h0.to(DEV))
    torch.autograd.backward((h, h_n), (dh.to(DEV), dh_n.to(DEV)))
    check(h.detach(), want["h"], memory, "halves")
    check(both.grad[..., :H], want["da"], memory, "halves da")
    check(both.grad[..., H:], want["db"], memory, "halves db")


@pytest.mark.parametrize("default", [torch.float64, torch.bfloat16, torch.float16], ids=str)
def test_states_are_float32_whatever_the_default_dtype(default):
    a, b, h0, s, dh, dh_n = make(70, 3, 40, torch.float32, "gated", seed=31, starts=True)
    for start in (h0, None):
        want = run(a, b, start, s, dh, dh_n, "gated")
        before = torch.get_default_dtype()
        torch.set_default_dtype(default)
        try:
            got = run(a, b, start, s, dh, dh_n, "gated")
        finally:
            torch.set_default_dtype(before)
        for k, v in want.items():
            if v is not None:
                assert got[k].dtype == v.dtype and torch.equal(got[k], v), k


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_overlapping_rows(dtype):
    """Windows of a signal: every step's row a few elements on, fewer steps than columns and more."""
    for T, H, hop in ((70, 64, 8), (5, 64, 1), (40, 33, 1), (20, 130, 1)):
        signal = make(T * hop + H + 8 - H % 8, 2, 1, dtype, "gated", seed=T)
        a, b = (t[:, :, 0].t().contiguous().to(DEV).unfold(1, H, hop)[:, :T].transpose(0, 1) for t in signal[:2])
        assert a.shape == (T, 2, H) and a.stride(0) == hop
        _, _, h0, _, dh, dh_n = make(T, 2, H, dtype, "gated", seed=T + 1)
        want, memory = truth(a, b, h0, None, dh, dh_n, "gated")
        z, x = a.detach().requires_grad_(True), b.detach().requires_grad_(True)
        h, h_n = call("gated")(z, x, h0.to(DEV))
        torch.autograd.backward([h, h_n], [dh.to(DEV), dh_n.to(DEV)])
        check_all(dict(h=h.detach(), h_n=h_n.detach(), da=z.grad, db=x.grad, dh0=None), want, memory, f"T={T} H={H}")
    import prlstm_b200 as P

    rows = a[:, 0]  # the single step on overlapping rows
    out, state = P.gated_recurrence_step(rows, b[:, 0], torch.zeros(T, H, device=DEV))
    want, memory = truth(rows[None], b[:, 0][None], torch.zeros(T, H), None, None, None, "gated")
    check(out, want["h"][0], memory, "step")
    check(state, want["h_n"], memory, "step state", torch.float32)


@pytest.mark.parametrize("zero", [0.0, -0.0])
def test_a_zero_coefficient_is_no_start(zero):
    """An infinite state times a zero of either sign is NaN, step by step; a start drops it."""
    T, H = 3000, 40
    a, b = torch.ones(T, 1, H, device=DEV), torch.zeros(T, 1, H, device=DEV)
    a[1000], b[2000] = zero, 3.0
    s = torch.zeros(T, 1, dtype=torch.bool, device=DEV)
    s[2000] = True
    h0 = torch.full((1, H), float("inf"), device=DEV)
    for starts in (s, torch.zeros_like(s)):
        h, h_n = call("linear")(a, b, h0, starts=starts)
        assert h[:1000].isposinf().all() and h[1000:2000].isnan().all()
        if starts is s:
            assert (h[2000:] == 3.0).all() and (h_n == 3.0).all()
        else:
            assert h[2000:].isnan().all() and h_n.isnan().all()


def walk(T, B, H, dtype, kind, seed):
    """Coefficients of either sign whose products leave float32's range while a
    state from 2^w_0 moves within it: its logarithm goes from w_t to w_{t+1}."""
    g = torch.Generator().manual_seed(seed)
    if kind == "up":
        w = torch.linspace(-110, 110, T + 1)
    elif kind == "down and up":
        w = 90 - 190 * (1 - (torch.linspace(-1, 1, T + 1)).abs())
    elif kind == "up and down":
        w = -90 + 190 * (1 - (torch.linspace(-1, 1, T + 1)).abs())
    elif kind == "saw":  # up by 3 a step for 60 steps, down by 60 a step
        at = torch.arange(T + 1) % 63
        w = torch.where(at <= 60, -90 + 3.0 * at, 90 - 60.0 * (at - 60))
    else:  # steps of up to 2^50 either way
        w = torch.empty(T + 1)
        w[0] = 0
        step = 100 * torch.rand(T, generator=g) - 50
        for t in range(T):
            w[t + 1] = w[t] + (step[t] if abs(float(w[t] + step[t])) < 100 else -step[t])
    a = torch.exp2((w[1:] - w[:-1]).double())[:, None, None] * torch.where(torch.rand(T, B, H, generator=g) < 0.5, -1.0, 1.0)
    return a.to(dtype), torch.exp2(w[0].double()).float()


GROWTH = [(32, 1, 64), (520, 1, 64), (2300, 1, 64), (2300, 1, 33), (900, 3, 70), (700, 40, 256), (2300, 1, 65)]


@pytest.mark.parametrize("starts", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("kind", ["up", "down and up", "up and down", "saw", "jumps"])
@pytest.mark.parametrize("shape", GROWTH, ids=str)
def test_coefficients_whose_products_leave_the_range(shape, kind, dtype, starts):
    """Each state is one product of t coefficients and the first state (no
    cancellation), so it is off by a unit 2^-24 a step, and so is the gradient
    that reaches a step from the end."""
    T, B, H = shape
    a, first = walk(T, B, H, dtype, kind, seed=T + H)
    h0 = first * (1 + torch.rand(B, H, generator=torch.Generator().manual_seed(1)))
    b = torch.zeros(T, B, H, dtype=dtype)
    s = None
    if starts:  # the sequence begins anew at a step or two, from b
        s = torch.zeros(T, B, dtype=torch.bool)
        for t in (T // 3, T // 3 + 20):
            s[t] = True
    want_h = torch.empty(T, B, H, dtype=torch.float64)
    state = h0.double()
    for t in range(T):
        state = a[t].double() * state
        if s is not None and bool(s[t].any()):
            b[t] = state.to(dtype)
            state = b[t].double()
        want_h[t] = state
    # backward on the coefficients taken from the last to the first, so that it walks the same way
    ra, rb = a.flip(0), torch.zeros_like(b)
    rs = None if s is None else s.flip(0)
    e, want_db, want_da = h0.double(), torch.empty_like(want_h), None
    for t in range(T - 1, -1, -1):
        want_db[t] = e
        e = ra[t].double() * e
        if rs is not None:
            e = torch.where(rs[t][:, None], 0.0, e)
    h, h_n = call("linear")(a.to(DEV), b.to(DEV), h0.to(DEV), starts=None if s is None else s.to(DEV))
    z, x = ra.to(DEV).requires_grad_(True), rb.to(DEV).requires_grad_(True)
    start = torch.zeros(B, H, device=DEV, requires_grad=True)
    _, end = call("linear")(z, x, start, starts=None if rs is None else rs.to(DEV))
    end.backward(h0.to(DEV))

    def same(got, want, what):
        got = got.double().cpu()
        tol = 2 * (T + 8) * 2.0 ** -24 + (UNIT[dtype] if what in ("h", "db") and dtype != torch.float32 else 0)
        worst = ((got - want).abs() / want.abs().clamp(min=2.0 ** -120)).max()
        assert float(worst) <= tol, f"{what}: {float(worst):.3e} > {tol:.3e}"

    same(h, want_h, "h")
    same(h_n, want_h[-1], "h_n")
    same(x.grad, want_db, "db")
    same(start.grad, e, "dh0")


@pytest.mark.parametrize("T,H", [(3000, 40), (3000, 33), (500, 4096)])
def test_states_that_overflow_are_infinite(T, H):
    """Growth past the range is an infinity from that step on, from a zero state nothing."""
    a, b = torch.full((T, 1, H), 2.0, device=DEV), torch.zeros(T, 1, H, device=DEV)
    h0 = torch.ones(1, H, device=DEV)
    h0[:, ::2] = 0
    h0[:, 1::4] = -1
    h, h_n = call("linear")(a, b, h0)
    assert (h[:, :, ::2] == 0).all() and (h_n[:, ::2] == 0).all()
    assert torch.equal(h[:126, 0, 1], torch.tensor([-2.0 ** n for n in range(1, 127)], device=DEV))
    assert h[127:, :, 1::4].isneginf().all() and h[127:, :, 3::4].isposinf().all()
    z, x = a.clone().requires_grad_(True), b.clone().requires_grad_(True)
    _, end = call("linear")(z, x)
    end.backward(h0)
    assert (x.grad[:, :, ::2] == 0).all() and x.grad[:T - 128, :, 3::4].isposinf().all()
    assert torch.equal(x.grad[T - 100:, 0, 3], torch.tensor([2.0 ** n for n in range(99, -1, -1)], device=DEV))
    # an infinite state outlasts a product of coefficients that is no float32
    h, _ = call("linear")(torch.full((T, 1, H), -0.5, device=DEV), b, torch.full((1, H), float("inf"), device=DEV))
    assert h.isinf().all() and bool((h[::2] < 0).all()) and bool((h[1::2] > 0).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("T,H", [(1, 32), (40, 33), (2100, 32), (2100, 34), (600, 4096)])
def test_nothing_passes_a_gate_that_is_shut(T, H, dtype):
    """Below float32's range a gate is 0: an input of 0 leaves 0, with and without starts in the run."""
    g = torch.Generator().manual_seed(T + H)
    x = torch.randn(T, 1, H, generator=g).to(dtype)
    x[torch.rand(T, 1, H, generator=g) < 0.2] = 0
    h0 = 100 * torch.randn(1, H, generator=g)
    z = torch.full((T, 1, H), -200.0, dtype=dtype)
    s = torch.rand(T, 1, generator=g) < 0.05
    for starts in (None, s.to(DEV)):
        h, h_n = call("gated")(z.to(DEV), x.to(DEV), h0.to(DEV), starts=starts)
        assert torch.equal(h.cpu(), x) and torch.equal(h_n.cpu(), x[-1].float())


@pytest.mark.parametrize("starts", [False, True])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", [(1, 1, 64), (5, 1, 64), (16, 1, 64), (48, 2, 66), (48, 2, 33), (700, 1, 64), (3000, 1, 64)], ids=str)
def test_gradient_through_small_gates(shape, dtype, starts):
    """A loss on the last state alone: what reaches the steps before a small gate is
    that gate's size, and as exact as anything else.  Each gate carries a few
    units 2^-24 of itself, so a gradient is off by those of all steps after it."""
    T, B, H = shape
    g = torch.Generator().manual_seed(T + H)
    z = 5 + 2 * torch.rand(T, B, H, generator=g)
    z[T // 2] = -20 + 12 * torch.rand(B, H, generator=g)
    z = z.to(dtype)
    x, h0 = torch.randn(T, B, H, generator=g).to(dtype), torch.randn(B, H, generator=g)
    dh_n = 1024 * torch.randn(B, H, generator=g)
    s = torch.zeros(T, B, dtype=torch.bool) if starts else None
    if starts and T > 16:
        s[T // 4] = True
    want, _ = truth(z, x, h0, s, None, dh_n, "gated")
    got = run(z, x, h0, s, None, dh_n, "gated")
    unit = (4 * T + 16) * 2.0 ** -24
    size = want["h"].abs().max() + x.double().abs().max() + h0.abs().max()  # of the difference that da holds
    f, om = torch.sigmoid(z.double()), torch.sigmoid(-z.double())
    e = want["db"] / om
    own = (UNIT[dtype] if dtype != torch.float32 else 0.0)
    for name, bound in (("dh0", unit * want["dh0"].abs()), ("db", (unit + own) * want["db"].abs() + TINY[dtype]),
                        ("da", unit * size * e.abs() * f * om + own * want["da"].abs() + TINY[dtype])):
        over = (got[name].double().cpu() - want[name]).abs() - bound - 2.0 ** -126
        assert float(over.max()) <= 0, f"{name}: {float(over.max()):.3e} over"


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("logit", [2.0, 0.0, -20.0])
@pytest.mark.parametrize("T,H", [(40, 32), (3000, 32), (3000, 33), (3000, 34), (600, 4096)])
def test_an_infinite_state_outlasts_any_number_of_gates(T, H, logit, dtype):
    """Times a gate above 0 it stays infinite, over runs and CTAs whose product of
    gates is no float32; a start ends it.  The gradient's chain is alike."""
    inf = float("inf")
    z = torch.full((T, 1, H), logit, dtype=dtype, device=DEV).requires_grad_(True)
    x = torch.ones(T, 1, H, dtype=dtype, device=DEV).requires_grad_(True)
    h0 = torch.full((1, H), inf, device=DEV)
    h0[:, ::3] = -inf
    start = torch.zeros(1, H, device=DEV).requires_grad_(True)
    for at in (None, T // 2 + 3):
        s = None
        if at is not None:
            s = torch.zeros(T, 1, dtype=torch.bool, device=DEV)
            s[at] = True
        h, h_n = call("gated")(z, x, h0, starts=s)
        end = T if at is None else at
        assert h[:end, :, ::3].isneginf().all() and h[:end, :, 1::3].isposinf().all()
        assert h[end:].isfinite().all() and (at is not None or torch.equal(h_n, h0))
        _, h_n = call("gated")(z, x, start, starts=s)
        dx, d0 = torch.autograd.grad(h_n, (x, start), h0)
        first = 0 if at is None else at
        assert dx[first:, :, ::3].isneginf().all() and dx[first:, :, 1::3].isposinf().all()
        assert not dx[:first].any() and (at is not None or torch.equal(d0, h0))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("form", ["gated", "linear"])
@pytest.mark.parametrize("T,H", [(1, 70), (40, 64), (2048, 64), (700, 4096), (2049, 33)])
def test_states_in_place(T, H, form, dtype):
    """The library's calls write the last state over the first, and dh0 over dh_n."""
    from prlstm_b200 import _lib
    from prlstm_b200 import _lm_functions as F

    a, b, h0, _, dh, dh_n = (None if t is None else t.to(DEV) for t in make(T, 1, H, dtype, form, seed=T))
    code, kind, index, strides = F._CODE[dtype], 0 if form == "gated" else 1, 0, (H, H)
    ckpt = torch.empty(_lib.function("hs_recurrence_checkpoint_bytes")(T, 1, H) // 4, dtype=torch.float32, device=DEV)
    status = _lib.host_status(0).timeout_ptr
    got = []
    for here in (False, True):
        first, grad = h0.clone(), dh_n.clone()
        last, d0 = (first, grad) if here else (torch.empty_like(h0), torch.empty_like(h0))
        h, da, db = torch.empty_like(a), torch.empty_like(a), torch.empty_like(a)
        F._call("hs_recurrence_forward", index, code, kind, a.data_ptr(), *strides, b.data_ptr(), *strides, first.data_ptr(), None, 0, 0,
                h.data_ptr(), *strides, last.data_ptr(), ckpt.data_ptr(), T, 1, H, status)
        F._call("hs_recurrence_backward", index, code, kind, a.data_ptr(), *strides, b.data_ptr(), *strides, ckpt.data_ptr(), 0,
                dh.data_ptr(), *strides, grad.data_ptr(), da.data_ptr(), *strides, db.data_ptr(), *strides, d0.data_ptr(), T, 1, H, status)
        got.append([t.clone() for t in (h, last, da, db, d0)])
    assert all(torch.equal(x, y) for x, y in zip(*got))
