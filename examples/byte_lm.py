"""A byte-level language model on the package's operators: trained on this
file's own text, then answering one byte at a time.

    python examples/byte_lm.py [--steps 300]

Training runs whole rows of bytes, several texts packed end to end into each:
embedding -> HeadStartLSTM in parallel mode -> a gated recurrence whose state
is dropped where a text starts -> projection to 256 logits -> log probability
of the next byte.  Answering runs the same layers for a single step from kept
states.  ``sequence_logprobs`` gives the same numbers either way.
"""

from __future__ import annotations

import argparse
import math
import os
import sys

import torch
import torch.nn as nn
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import prlstm_b200 as P  # noqa: E402


class ByteModel(nn.Module):
    def __init__(self, width: int = 256, dtype=torch.float32):
        super().__init__()
        self.width = width
        self.table = nn.Parameter(torch.randn(256, width, dtype=dtype) / math.sqrt(width))
        self.lstm = P.HeadStartLSTM(width, width, parallel=True).to(dtype)
        self.gates = nn.Linear(width, 2 * width, dtype=dtype)
        self.head = nn.Linear(width, 256, dtype=dtype)
        with torch.no_grad():
            self.gates.bias[:width] = torch.linspace(-1, 4, width)  # memories of a step to some fifty

    def logits(self, tokens, starts=None, state=None):
        """tokens [T, B] -> logits [T, B, 256] and the state after the last."""
        x = P.embedding(tokens, self.table, scale=math.sqrt(self.width))
        lstm_state, h0 = (None, None) if state is None else state
        y, lstm_state = self.lstm(x, lstm_state)
        z, v = self.gates(x + y).chunk(2, dim=-1)  # taken as the slices they are
        h, h_n = P.gated_recurrence(z, v, h0, starts=starts)
        return self.head(x + y + h), (lstm_state, h_n)

    @torch.no_grad()
    def step(self, token, state):
        """One byte for each of B running texts: token [B] -> logits [B, 256].
        The gated state advances in place."""
        x = P.embedding(token, self.table, scale=math.sqrt(self.width))
        lstm_state, h = state
        y, lstm_state = self.lstm(x[None], lstm_state)
        y = y[0]
        z, v = self.gates(x + y).chunk(2, dim=-1)
        out, _ = P.gated_recurrence_step(z, v, h, out_state=h)
        return self.head(x + y + out), (lstm_state, h)

    def fresh_state(self, batch):
        dev, dt = self.table.device, self.table.dtype
        zero = torch.zeros(1, batch, self.width, device=dev, dtype=dt)
        return (zero, zero), torch.zeros(batch, self.width, device=dev)


def batch_of(text, rows, length, generator):
    """`rows` rows of `length` bytes cut out of the text, two pieces packed
    into each: inputs and next bytes [T, B] (no prediction across the seam),
    starts [T, B]."""
    half = length // 2
    at = torch.randint(0, len(text) - half - 1, (2, rows), generator=generator)
    take = at[:, None, :] + torch.arange(half)[None, :, None]
    inputs, targets = text[take].reshape(2 * half, rows), text[take + 1].reshape(2 * half, rows)
    starts = torch.zeros(2 * half, rows, dtype=torch.bool)
    starts[half] = True
    return inputs, targets, starts


def sequence_logprobs(model, tokens):
    """Log probabilities of bytes 1.. of tokens [T, B], read at once."""
    logits, _ = model.logits(tokens[:-1])
    return P.token_logprobs(logits, tokens[1:]).logprob


def train(model, text, steps, rows=32, length=256, lr=3e-3, seed=0, report=50):
    g = torch.Generator().manual_seed(seed)
    opt = torch.optim.AdamW(model.parameters(), lr=lr)
    dev, losses = model.table.device, []
    for n in range(steps):
        inputs, targets, starts = (t.to(dev) for t in batch_of(text, rows, length, g))
        logits, _ = model.logits(inputs, starts)
        r = P.token_logprobs(logits, targets)
        loss = -r.logprob.mean()
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
        losses.append(loss.detach())
        if report and n % report == 0:
            print(f"step {n}: loss {loss.item():.3f}, entropy {r.entropy.mean().item():.3f}", flush=True)
    return torch.stack(losses).tolist()


@torch.no_grad()
def answer(model, prompt: bytes, length: int, temperature: float = 0.7, seed: int = 0):
    """`length` sampled bytes after the prompt, with the log probability and
    the three most likely alternatives of each."""
    dev = model.table.device
    g = torch.Generator(device=dev).manual_seed(seed)
    tokens = torch.tensor(list(prompt), device=dev)[:, None]
    logits, state = model.logits(tokens, state=model.fresh_state(1))
    logits, out = logits[-1], []
    for _ in range(length):
        noise = torch.rand(logits.shape, device=dev, generator=g).log_().neg_().log_().neg_()
        token = (logits.float() / temperature + noise).argmax(-1)
        r = P.token_logprobs(logits, token, top=3, temperature=temperature)
        out.append((token, r.logprob, r.top_index, r.top_logprob))
        logits, state = model.step(token, state)
    return [(int(t), float(lp), i[0].tolist(), lps[0].tolist()) for t, lp, i, lps in out]


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--steps", type=int, default=300)
    a = ap.parse_args()
    torch.manual_seed(0)
    with open(os.path.abspath(__file__), "rb") as f:
        text = torch.frombuffer(bytearray(f.read()), dtype=torch.uint8).long()
    model = ByteModel().cuda()
    train(model, text, a.steps)
    P.check_device_status()
    said = answer(model, b"def ", 60)
    print(repr(bytes([t for t, *_ in said])))
    for t, lp, ids, lps in said[:5]:
        print(f"{chr(t)!r} {lp:.2f}   " + ", ".join(f"{chr(i)!r} {v:.2f}" for i, v in zip(ids, lps)))


if __name__ == "__main__":
    main()
