"""The operators together, as the byte-level example uses them: training
lowers the loss, reading a text at once and byte by byte gives the same log
probabilities, and a whole training step can be captured in a CUDA graph."""

import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = torch.device("cuda", 0)


@pytest.fixture(scope="module")
def lm():
    path = os.path.join(ROOT, "examples", "byte_lm.py")
    spec = importlib.util.spec_from_file_location("byte_lm", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.fixture(scope="module")
def text():
    return torch.frombuffer(bytearray(b"the quick brown fox jumps over the lazy dog. " * 60), dtype=torch.uint8).long()


def test_training_learns_the_text(lm, text):
    torch.manual_seed(1)
    model = lm.ByteModel(128).to(DEV)
    losses = lm.train(model, text, 60, rows=16, length=128, report=0)
    assert all(v == v for v in losses)
    # from about ln 256 = 5.5 to below 1: the text repeats every 45 bytes
    assert losses[0] > 4 and sum(losses[-5:]) / 5 < 1.0, (losses[0], losses[-5:])
    said = lm.answer(model, b"the quick ", 20, temperature=0.1)
    assert len(said) == 20 and all(lps[0] >= lps[1] >= lps[2] and lp <= 0 for _, lp, _, lps in said)


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2e-5), (torch.bfloat16, 0.15)])
def test_whole_sequences_and_single_steps_agree(lm, text, dtype, tol):
    """float32: the paths differ by the order of float32 sums, some 1e-6 of
    logits of a few units.  bfloat16: activations are rounded to 2^-8 at each layer in
    either path, to different sides at most, over logits of a few units."""
    torch.manual_seed(2)
    model = lm.ByteModel(128, dtype).to(DEV)
    tokens = torch.stack([text[i:i + 40] for i in (0, 17, 100)], 1).to(DEV)
    with torch.no_grad():
        at_once = lm.sequence_logprobs(model, tokens)
        state, rows = model.fresh_state(3), []
        for t in range(39):
            logits, state = model.step(tokens[t], state)
            rows.append(lm.P.token_logprobs(logits, tokens[t + 1]).logprob)
    assert (at_once - torch.stack(rows)).abs().max() < tol


def test_captured_training_step_equals_eager(lm, text):
    """Embedding, gated recurrence and loss, forward and backward, replayed from
    a CUDA graph on new inputs: the same bits as eager calls."""
    P = lm.P
    g = torch.Generator().manual_seed(3)
    table = (torch.randn(256, 64, generator=g) / 8).to(DEV).requires_grad_(True)
    w = (torch.randn(128, 64, generator=g) / 8).to(DEV).requires_grad_(True)
    head = (torch.randn(256, 64, generator=g) / 8).to(DEV).requires_grad_(True)

    def step(inputs, targets, starts):
        x = P.embedding(inputs, table, scale=8.0)
        z, v = torch.nn.functional.linear(x, w).chunk(2, -1)
        h, h_n = P.gated_recurrence(z, v, starts=starts)
        r = P.token_logprobs(torch.nn.functional.linear(h, head), targets, top=3)
        loss = -(r.logprob + 0.01 * r.entropy).mean()
        return (loss.detach(), h_n.detach(), r.top_index) + torch.autograd.grad(loss, (table, w, head))

    batches = [tuple(t.to(DEV) for t in lm.batch_of(text, 6, 200, g)) for _ in range(3)]
    want = [[t.clone() for t in step(*b)] for b in batches]
    static = [t.clone() for t in batches[0]]
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(side):
        step(*static)
    torch.cuda.current_stream(DEV).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*static)
    for b, expect in zip(batches, want):
        for s, t in zip(static, b):
            s.copy_(t)
        graph.replay()
        torch.cuda.synchronize(DEV)
        for i, (a, e) in enumerate(zip(out, expect)):
            assert torch.equal(a, e), i
    P.check_device_status()
    del graph
