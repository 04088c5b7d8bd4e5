"""What the language-model operators' sources have to hold to and a run would
show by chance only (CPU only)."""

import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "prlstm_b200", "csrc")


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return f.read()


@pytest.mark.parametrize("name", ["gated_recurrence.cu", "token_logprobs.cu", "embedding.cu"])
def test_warps_meet_before_aligned_cluster_barriers(name):
    """An aligned barrier is one instruction of the whole warp: whatever stands
    before it, the lanes are brought together first."""
    lines = source(name).splitlines()
    at = [i for i, line in enumerate(lines) if re.search(r"barrier\.cluster\.\w+\.\w+\.aligned", line)]
    assert at
    for i in at:
        assert "__syncwarp();" in lines[i - 1], f"{name}:{i + 1}"


def test_counters_are_zero_before_any_lane_counts():
    """The finder of a row's alternatives: one lane clears the counters, others
    add to them; between the two memory is ordered for a warp per row (votes do not
    order it) and for a CTA per row."""
    text = source("token_logprobs.cu")
    clear = text.index("f.nfound = f.nchosen = f.nkept = 0;")
    between = text[clear:text.index("atomicAdd(&f.", clear)]
    assert "if (W == 1) __syncwarp();" in between and "__syncthreads();" in between


def test_stores_precede_bulk_copies_into_the_same_place():
    """The rows' copies write some bytes by the lanes themselves; a later wave's
    bulk copy goes into the same bytes by another path, which only a fence orders."""
    text = source("gated_recurrence.cu")
    body = text[text.index("HS_DEV unsigned copy_row("):]
    body = body[:body.index("\n}\n")]
    stores, fence = body.rindex("st.shared.u16"), body.find("fence_async();")
    assert stores < fence < body.index("cp.async.bulk.shared::cluster")


@pytest.mark.parametrize("kernel,store", [("rec_fwd_kernel", "p.h_n[row"), ("rec_bwd_kernel", "p.dh0[row")])
def test_last_states_are_written_after_all_have_read_the_first(kernel, store):
    """h_n may be h0 (dh0 may be dh_n), which every CTA of a cluster reads: the store
    stands behind the barrier that ends the cluster's work."""
    text = source("gated_recurrence.cu")
    body = text[text.index(kernel + "(const __grid_constant__"):]
    at = body.index(store)
    assert body.rindex("cluster_arrive();", 0, at) < body.rindex("cluster_wait();", 0, at) < at
    assert "for (int w = 0; w < waves" not in body[body.rindex("cluster_arrive();", 0, at):at]
