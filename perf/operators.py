"""Measured cases of the language-model operators around the scan: the gated
linear recurrence, the embedding with its gradient, and the log probabilities
of given tokens.

Each case names one call (or one training step: forward and gradient) at one
size.  ``run`` computes it either in elementary torch operations in 32 bits,
rounded once at the end (``own`` false), or through this package's entry points
(``own`` true); ``exact`` computes it from the definition in 64 bits.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
DEV = "cuda"
LARGEST = 1 << 27  # values of one of the large tensors of the largest cases


def listed():
    """Recurrence: op "recurrence", T x B x H, form "gated" (gate logits z and
    values x) or "linear" (coefficients given), documents packed into rows.
    Embedding: op "embedding", N tokens of a V x D table.  Log probabilities:
    op "logprobs", N rows of V logits, the `top` best alternatives."""
    return [
        # one token for each of 64 running requests: what a server pays per token and layer
        dict(name="step 64x1024 bf16", op="recurrence", mode="step", form="gated", dtype="bf16", T=1, B=64, H=1024, starts=False),
        # the short training shape of this repository's scan (T=128, B=32, H=256), many small steps
        dict(name="train 128x32x256 f32", op="recurrence", mode="train", form="gated", dtype="f32", T=128, B=32, H=256, starts=False),
        # odd sizes, signed coefficients given by the caller, rows not a multiple of any vector
        dict(name="train 1003x3x333 linear f16", op="recurrence", mode="train", form="linear", dtype="f16", T=1003, B=3, H=333, starts=True),
        # the long training shape (T=16384, H=1024), documents packed end to end
        dict(name="train 16384x8x1024 bf16", op="recurrence", mode="train", form="gated", dtype="bf16", T=16384, B=8, H=1024, starts=True),
        # one long prompt read in before the first answer token
        dict(name="prompt 16384x1x1024 f32", op="recurrence", mode="forward", form="gated", dtype="f32", T=16384, B=1, H=1024, starts=False),
        # the next token of 64 requests
        dict(name="embed 64 of 32000x512 bf16", op="embedding", mode="forward", dtype="bf16", N=64, V=32000, D=512),
        # one training micro-batch (256 steps x 32 sequences)
        dict(name="embed train 8192 f32", op="embedding", mode="train", dtype="f32", N=8192, V=32000, D=512),
        # a large vocabulary and a long batch
        dict(name="embed train 131072 bf16", op="embedding", mode="train", dtype="bf16", N=131072, V=131072, D=1024),
        # answers of 24 requests with the 20 best alternatives, a grammar masking most of the vocabulary
        dict(name="logprobs 24x131072 top20 f32", op="logprobs", mode="forward", dtype="f32", N=24, V=131072, top=20, masked=True),
        # scoring given text under a vocabulary of odd size
        dict(name="score 2047x50021 top5 bf16", op="logprobs", mode="forward", dtype="bf16", N=2047, V=50021, top=5, masked=False),
        # a byte-level model's training step
        dict(name="loss 4096x256 f32", op="logprobs", mode="train", dtype="f32", N=4096, V=256, top=0, masked=False),
        # a training batch: log probabilities and entropy with the gradient of all logits
        dict(name="loss 16384x32000 bf16", op="logprobs", mode="train", dtype="bf16", N=16384, V=32000, top=0, masked=False),
    ]


def draw(rng: random.Random):
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op, dtype = rng.choice(("recurrence", "embedding", "logprobs")), rng.choice(("f32", "bf16", "f16"))
    if op == "recurrence":
        B, H = size(1, 96), size(8, 2048)
        mode = rng.choice(("step", "forward", "train", "train"))
        T = 1 if mode == "step" else min(size(2, 16384), max(2, LARGEST // (B * H)))
        return dict(op=op, mode=mode, form=rng.choice(("gated", "linear")), dtype=dtype, T=T, B=B, H=H, starts=mode != "step" and rng.random() < 0.5)
    if op == "embedding":
        D = size(16, 2048)
        return dict(op=op, mode=rng.choice(("forward", "train", "train")), dtype=dtype, N=min(size(1, 131072), LARGEST // D),
                    V=min(size(200, 131072), LARGEST // D), D=D)
    V = size(60, 200000)
    mode = rng.choice(("forward", "train"))
    return dict(op=op, mode=mode, dtype=dtype, N=max(1, min(size(1, 16384), 2 * LARGEST // V)), V=V,
                top=rng.randint(0, 20) if mode == "forward" else 0, masked=rng.random() < 0.3)


# ------------------------------------------------------------------ inputs
def _tokens(n, vocab, g):
    """Token ids with the skew of text: the k-th commonest token about 1/k as
    frequent as the first (log-uniform ranks), ids in no order of frequency."""
    u = torch.rand(n, device=DEV, generator=g, dtype=torch.float64)
    rank = torch.exp(u * math.log(vocab + 1)).long().clamp_(1, vocab) - 1
    return (rank * 48271 + 11) % vocab  # the multiplier is a prime above every vocabulary's factors


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, device=DEV, generator=g)

    s = dict(case=dict(case))
    train = case["mode"] == "train"
    if case["op"] == "recurrence":
        T, B, H = case["T"], case["B"], case["H"]
        if case["form"] == "gated":
            # forget gates from about 0.3 to 0.9995: memories of a step to thousands of steps
            s["a"], s["b"] = (1.8 * normal(T, B, H) + 2.5).to(dt), normal(T, B, H).to(dt)
        else:
            s["a"], s["b"] = torch.tanh(normal(T, B, H) + 1.5).to(dt), normal(T, B, H).to(dt)
        s["h0"] = normal(B, H)
        s["starts"] = torch.rand(T, B, device=DEV, generator=g) < 1 / 400 if case["starts"] else None
        if case["mode"] == "step":
            s["a"], s["b"] = s["a"][0], s["b"][0]
        if train:
            s["dh"], s["dh_n"] = normal(T, B, H).to(dt), normal(B, H)
            for k in ("a", "b", "h0"):
                s[k].requires_grad_(True)
    elif case["op"] == "embedding":
        N, V, D = case["N"], case["V"], case["D"]
        s["weight"] = (normal(V, D) / math.sqrt(D)).to(dt)
        s["tokens"] = _tokens(N, V, g)
        s["scale"] = math.sqrt(D)
        s["padding_idx"] = int(s["tokens"][0]) if N > 1 else None
        if train:
            s["dout"] = normal(N, D).to(dt)
            s["weight"].requires_grad_(True)
    else:
        N, V = case["N"], case["V"]
        x = 2.0 * normal(N, V)
        s["tokens"] = _tokens(N, V, g)
        if case["masked"]:  # a grammar leaves about a tenth of the vocabulary; the answer is among it
            keep = torch.rand(N, V, device=DEV, generator=g) < 0.1
            keep.scatter_(1, s["tokens"][:, None], True)
            x.masked_fill_(~keep, -math.inf)
            del keep
        s["logits"] = x.to(dt)
        s["temperature"] = 0.8
        if train:
            s["tokens"][torch.rand(N, device=DEV, generator=g) < 0.05] = -100  # padding
            s["dlogprob"], s["dentropy"] = normal(N), 0.1 * normal(N)
            s["logits"].requires_grad_(True)
    return s


# ------------------------------------------------------------------ the plain form
def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along the first axis from h_{-1} = 0 by doubling:
    ceil(log2 T) passes of elementwise products and sums over whole tensors."""
    d = 1
    while d < a.shape[0]:
        b = torch.cat((b[:d], torch.addcmul(b[d:], a[d:], b[:-d])))
        a = torch.cat((a[:d], a[d:] * a[:-d]))
        d *= 2
    return b


def _plain_recurrence(s):
    case, dt = s["case"], s["a"].dtype
    a, x, h0 = s["a"].detach().float(), s["b"].detach().float(), s["h0"].detach()
    if case["mode"] == "step":
        a, x = a[None], x[None]
    gated = case["form"] == "gated"
    f = torch.sigmoid(a) if gated else a
    b = (1 - f) * x if gated else x
    keep = f if s["starts"] is None else f.masked_fill(s["starts"][:, :, None], 0)
    b0 = torch.cat((torch.addcmul(b[:1], keep[:1], h0[None]), b[1:]))
    h = _scan(keep, b0)
    h_n = h[-1].clone()
    if case["mode"] == "step":
        return {"h": h[0].to(dt), "h_n": h_n}
    if case["mode"] == "forward":
        return {"h": h.to(dt), "h_n": h_n}
    g = s["dh"].to(torch.float32, copy=True)
    g[-1] += s["dh_n"]
    after = torch.cat((keep[1:], torch.zeros_like(keep[:1])))
    e = _scan(after.flip(0), g.flip(0)).flip(0)
    before = torch.cat((h0[None], h[:-1]))
    if s["starts"] is not None:
        before = before.masked_fill(s["starts"][:, :, None], 0)
    da = e * (before - x) * f * (1 - f) if gated else e * before
    db = e * (1 - f) if gated else e
    return {"h": h.to(dt), "h_n": h_n, "da": da.to(dt), "db": db.to(dt), "dh0": keep[0] * e[0]}


def _plain_embedding(s):
    w, tok, dt = s["weight"].detach(), s["tokens"], s["weight"].dtype
    out = (w[tok].float() * s["scale"]).to(dt)
    if s["case"]["mode"] == "forward":
        return {"out": out}
    dout = s["dout"].float() * s["scale"]
    if s["padding_idx"] is not None:
        dout = dout.masked_fill((tok == s["padding_idx"])[:, None], 0)
    dw = torch.zeros(w.shape, device=DEV).index_add_(0, tok, dout)
    return {"out": out, "dweight": dw.to(dt)}


def _plain_logprobs(s):
    case, top = s["case"], s["case"]["top"]
    raw, tok = s["logits"].detach(), s["tokens"]
    x = raw.float() / s["temperature"]
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(1, keepdim=True)
    lse = m + torch.log(total)
    p, lp = e / total, x - lse
    plp = torch.where(p > 0, p * lp, 0)
    entropy = -plp.sum(1)
    live = tok != -100
    at = torch.where(live, tok, 0)[:, None]
    out = {"logprob": torch.where(live, lp.gather(1, at)[:, 0], 0), "entropy": torch.where(live, entropy, 0)}
    if top:
        # order by value, then the lowest index: both in one whole number
        k = min(top, case["V"])
        bits = raw.float().add(0.0).view(torch.int32).long()
        key = torch.where(bits < 0, -1 - (bits & 0x7FFFFFFF), bits) << 32
        key += torch.arange(case["V"] - 1, -1, -1, device=DEV)
        idx = case["V"] - 1 - (torch.topk(key, k, dim=1).values & 0xFFFFFFFF)
        out["top_index"], out["top_logprob"] = idx, lp.gather(1, idx)
    if case["mode"] == "train":
        g, ge = s["dlogprob"][:, None], s["dentropy"][:, None]
        d = -p * g - ge * (plp + p * entropy[:, None])
        d.scatter_add_(1, at, g)
        out["dlogits"] = torch.where(live[:, None], d / s["temperature"], 0).to(raw.dtype)
    return out


# ------------------------------------------------------------------ the package's entry points
def _own(s):
    import prlstm_b200 as P

    case, train = s["case"], s["case"]["mode"] == "train"
    if case["op"] == "recurrence":
        gated = case["form"] == "gated"
        if case["mode"] == "step":
            h, h_n = (P.gated_recurrence_step if gated else P.linear_recurrence_step)(s["a"], s["b"], s["h0"])
            return {"h": h, "h_n": h_n}
        h, h_n = (P.gated_recurrence if gated else P.linear_recurrence)(s["a"], s["b"], s["h0"], starts=s["starts"])
        if not train:
            return {"h": h, "h_n": h_n}
        da, db, dh0 = torch.autograd.grad((h, h_n), (s["a"], s["b"], s["h0"]), (s["dh"], s["dh_n"]))
        return {"h": h, "h_n": h_n, "da": da, "db": db, "dh0": dh0}
    if case["op"] == "embedding":
        out = P.embedding(s["tokens"], s["weight"], scale=s["scale"], padding_idx=s["padding_idx"])
        if not train:
            return {"out": out}
        (dw,) = torch.autograd.grad(out, s["weight"], s["dout"])
        return {"out": out, "dweight": dw}
    r = P.token_logprobs(s["logits"], s["tokens"], top=min(case["top"], case["V"]), temperature=s["temperature"])
    out = {"logprob": r.logprob, "entropy": r.entropy}
    if case["top"]:
        out["top_index"], out["top_logprob"] = r.top_index, r.top_logprob
    if train:
        (out["dlogits"],) = torch.autograd.grad((r.logprob, r.entropy), s["logits"], (s["dlogprob"], s["dentropy"]))
    return out


def run(state):
    if own:
        return _own(state)
    return {"recurrence": _plain_recurrence, "embedding": _plain_embedding, "logprobs": _plain_logprobs}[state["case"]["op"]](state)


# ------------------------------------------------------------------ bytes and operations
def work(case):
    es, train = BYTES[case["dtype"]], case["mode"] == "train"
    if case["op"] == "recurrence":
        n, state = case["T"] * case["B"] * case["H"], case["B"] * case["H"]
        # z, x, dh in; h, dz, dx out (forward alone: z, x in, h out); the states in 32 bits
        return {"bytes": n * es * (6 if train else 3) + state * 4 * (4 if train else 2), "flops": n * (24 if train else 8)}
    if case["op"] == "embedding":
        n, rows = case["N"] * case["D"], min(case["N"], case["V"]) * case["D"]
        b = case["N"] * 8 + (rows + n) * es
        return {"bytes": b + ((n + case["V"] * case["D"]) * es if train else 0), "flops": n * (2 if train else 1)}
    n = case["N"] * case["V"]
    b = n * es * (2 if train else 1) + case["N"] * (16 + 12 * case["top"] + (8 if train else 0))
    return {"bytes": b, "flops": n * (12 if train else 6)}


# ------------------------------------------------------------------ 64 bits, from the definition
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"recurrence": _exact_recurrence, "embedding": _exact_embedding, "logprobs": _exact_logprobs}[case["op"]](case, s)


def _exact_recurrence(case, s):
    T, B, H = case["T"], case["B"], case["H"]
    a, x = s["a"].double().view(T, B, H), s["b"].double().view(T, B, H)
    gated = case["form"] == "gated"
    cut = None if s["starts"] is None else (~s["starts"]).double()[:, :, None]
    f = 1 / (1 + torch.exp(-a)) if gated else a
    one_minus = 1 / (1 + torch.exp(a)) if gated else None
    keep = f if cut is None else f * cut
    h = one_minus * x if gated else x.clone()
    state = s["h0"].double()
    for t in range(T):  # step by step
        h[t].addcmul_(keep[t], state)
        state = h[t]
    out = {"h": h, "h_n": h[-1].clone()}
    if case["mode"] == "step":
        return {"h": h[0], "h_n": h[-1].clone()}
    if case["mode"] == "train":
        e = s["dh"].double()
        e[-1] += s["dh_n"].double()
        for t in range(T - 2, -1, -1):
            e[t].addcmul_(keep[t + 1], e[t + 1])
        before = torch.empty_like(h)
        before[0], before[1:] = s["h0"].double(), h[:-1]
        if cut is not None:
            before *= cut
        out["dh0"] = keep[0] * e[0]
        out["da"] = e * (before - x) * f * one_minus if gated else e * before
        out["db"] = e * one_minus if gated else e
    return out


def _exact_embedding(case, s):
    w, tok = s["weight"].double(), s["tokens"]
    out = {"out": w.index_select(0, tok) * s["scale"]}
    if case["mode"] == "train":
        # sums of runs of the sorted tokens as differences of running sums, in
        # pieces of columns (64 bits hold the differences to about 1e-13)
        order = torch.argsort(tok, stable=True)
        if s["padding_idx"] is not None:
            order = order[tok[order] != s["padding_idx"]]
        at = tok[order]
        ends = torch.searchsorted(at, torch.arange(case["V"], device=DEV), right=True)
        dw = torch.zeros(case["V"], case["D"], device=DEV, dtype=torch.float64)
        for c in range(0, case["D"], 128):
            run = torch.zeros(len(order) + 1, min(128, case["D"] - c), device=DEV, dtype=torch.float64)
            torch.cumsum(s["dout"][:, c:c + 128][order].double() * s["scale"], 0, out=run[1:])
            upto = run[ends]
            dw[:, c:c + 128] = upto
            dw[1:, c:c + 128] -= upto[:-1]
        out["dweight"] = dw
    return out


def _exact_logprobs(case, s):
    N, V, top, T = case["N"], case["V"], min(case["top"], case["V"]), s["temperature"]
    rows = max(1, (1 << 25) // V)
    parts = []
    for r in range(0, N, rows):
        raw, tok = s["logits"][r:r + rows].double(), s["tokens"][r:r + rows]
        lp = torch.log_softmax(raw / T, 1)
        p = lp.exp()
        ent = torch.special.entr(p).sum(1)
        live = tok >= 0
        at = tok.clamp(min=0)
        i = torch.arange(len(tok), device=DEV)
        part = {"logprob": lp[i, at] * live, "entropy": ent * live}
        if top:
            order = torch.sort(raw, dim=1, descending=True, stable=True).indices[:, :top]
            part["top_index"], part["top_logprob"] = order, lp.gather(1, order)
        if case["mode"] == "train":
            g, ge = s["dlogprob"][r:r + rows].double(), s["dentropy"][r:r + rows].double()
            d = -p * g[:, None] + ge[:, None] * (torch.special.entr(p) - p * ent[:, None])
            d[i, at] += g
            part["dlogits"] = d * live[:, None] / T
        parts.append(part)
    return {k: torch.cat([q[k] for q in parts]) for k in parts[0]}
