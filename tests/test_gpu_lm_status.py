"""The status words of the language-model operators in pinned host memory."""

import os
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = torch.device("cuda", 0)


def child(code):
    """Runs `code` in a process of its own, where no operator has been called yet."""
    r = subprocess.run([sys.executable, "-c", "import torch\nimport prlstm_b200 as P\n" + code], cwd=ROOT, capture_output=True,
                       text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    return r.stdout


def test_first_call_under_a_cuda_default_device():
    child("""
torch.set_default_device("cuda")
z = torch.randn(4, 2, 8)
h, h_n = P.gated_recurrence(z, z)
assert torch.equal(h[-1], h_n)
assert P.embedding(torch.tensor([1, 0]), z[0]).shape == (2, 8)
assert P.token_logprobs(z[0], torch.tensor([1, 2]), top=2).top_index.shape == (2, 2)
P.check_device_status()
""")


def test_clearing_waits_for_every_stream():
    """A bad id still on its way on another stream is cleared, too, not reported by the next call."""
    import prlstm_b200 as P

    table, good, bad = torch.randn(10, 8, device=DEV), torch.tensor([1], device=DEV), torch.tensor([99], device=DEV)
    P.embedding(good, table)
    P.clear_device_status()
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream(DEV))
    try:
        with torch.cuda.stream(side):
            torch.cuda._sleep(200_000_000)  # about a tenth of a second
            P.embedding(bad, table)
        P.clear_device_status()
        side.synchronize()
        P.embedding(good, table)
        P.check_device_status()
    finally:
        side.synchronize()
        P.clear_device_status()
