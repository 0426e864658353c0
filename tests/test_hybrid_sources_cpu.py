"""What no run on a GPU shows: properties of the hybrid-stack kernels held by reading their sources, and refusals of sizes that no GPU holds."""
import ctypes
import os
import re

import pytest
import torch

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "log-linear-attention_b200", "csrc")


def kernels(name):
    """{kernel: its body without comments} of a source file."""
    with open(os.path.join(CSRC, name)) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    found = {}
    for m in re.finditer(r"__global__[^;{]*?\b(\w+_kernel)\(", text):
        at = text.index("{", m.end())
        depth, end = 0, at
        while True:
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            end += 1
            if depth == 0:
                break
        found[m.group(1)] = text[at:end]
    return found


WINDOW = [("window_fwd_tc.cu", "window_fwd_tc_kernel"), ("window_bwd_tc.cu", "window_dq_tc_kernel"), ("window_bwd_tc.cu", "window_dkv_tc_kernel")]


@pytest.mark.parametrize("file,kernel", WINDOW)
def test_copies_and_products_end_before_the_cta_after_a_wait_that_gave_up(file, kernel):
    """Any thread may give up until the CTA's last barrier.  Only behind it is the abort flag final: there, and not in front of it, the copies that were issued and the products are waited for.  (In front of it
    the thread that issues them may look before another gives up, and the next CTA's shared memory would be written to.)"""
    body = kernels(file)[kernel]
    last = body.rindex("__syncthreads();")
    before, behind = body[:last], body[last:]
    assert not re.search(r"if \(\*abort_flag\)", before), "a decision on a flag that may still be set"
    assert re.search(r"if \(\*abort_flag\)", behind) and "end_products(" in behind
    assert len(re.findall(r"\.drain\(|mbar_wait\(full", behind)) >= (1 if "fwd" in kernel else 2)


@pytest.mark.parametrize("file,kernel", WINDOW)
def test_the_last_arrival_of_products_is_waited_for(file, kernel):
    """An arrival that nobody waits for may come when the CTA's shared memory is another's: the issuing warp's last commit is one that the rows wait for."""
    body = kernels(file)[kernel]
    issue = body[body.index("warp == MMA_WARP) {\n            const uint32_t lead"):body.index("SM::regs_rows()")]
    if "fwd" in kernel:                                  # (commits in a loop, whose last round has those for the rows alone)
        assert re.findall(r"(.*)commit_lead\(lead, empty", issue) == ["                if (i > 0 && i < count) umma::", "                if (i < count) umma::"]
    else:
        assert re.findall(r"commit_lead\(lead, (\w+)", issue)[-1] == "barDone"


@pytest.fixture(scope="module")
def pkg():
    import __graft_entry__ as ge
    ge.build()
    import hattention_b200
    return hattention_b200


@pytest.mark.parametrize("shape", [(1, 2 ** 32 + 5, 1), (2 ** 31, 1, 1), (1, 1, 2 ** 32 + 64)])
def test_recurrence_sizes_that_an_int_does_not_hold_are_refused(pkg, shape):
    """(Such a size reached the kernels modulo 2^32, which then left most of the output as it was.)"""
    x = torch.zeros(1, 1, 1, dtype=torch.bfloat16).expand(shape)
    with pytest.raises(ValueError, match="2\\^31"):
        pkg.gated_recurrence(x, x)
    if shape[1] == 1:
        x = x[:, 0]
        with pytest.raises(ValueError, match="2\\^31"):
            pkg.gated_recurrence_step(torch.zeros(1, 1).expand(x.shape), x, x)


def test_rows_whose_columns_an_int_does_not_count_are_refused(pkg):
    """The kernels for long rows count columns in ints, a stride of up to 256 past the end: rows of nearly 2^31 values would be read in front of their start."""
    from hattention_b200 import _lib
    lib, ok, null = _lib.lib(), ctypes.c_void_p(4096), ctypes.c_void_p(0)
    for N in (2 ** 30 + 1, 2 ** 31 - 1):
        assert lib.llattn_layer_norm_bwd_workspace_bytes(1, N) == 0
        assert lib.llattn_layer_norm_bwd(ok, 0, null, 1, ok, ok, ok, ok, null, null, null, 0, 1, N, null) == -1
        assert lib.llattn_layer_norm_fwd(null, 0, null, null, 1, ok, null, null, 1e-5, 1, N, null) == -1
        with pytest.raises(ValueError, match="2\\^30"):
            pkg.layer_norm(torch.zeros(1, dtype=torch.bfloat16).expand(N))
    assert lib.llattn_layer_norm_bwd_workspace_bytes(1, 2 ** 30) == 2 ** 33


def test_window_entries_take_16_byte_boundaries(pkg):
    """As those of the other operators: all loads and stores are of 16 bytes at most.  (A workspace that is too small is found behind the alignment, before a device is touched.)"""
    from hattention_b200 import _lib
    lib, P = _lib.lib(), ctypes.c_void_p
    ok, at16, odd, sizes = P(4096), P(4096 + 16), P(4096 + 8), (1, 8, 4, 2, 64, 4, 0, 1.0, P(0))
    fwd = lambda o, stats: lib.llattn_window_fwd(ok, ok, ok, o, stats, ok, 0, *sizes)
    assert fwd(at16, at16) == -5 and fwd(odd, ok) == -9 and fwd(ok, odd) == -9
    bwd = lambda stats, dq, dk, dv: lib.llattn_window_bwd(ok, ok, ok, ok, stats, ok, dq, dk, dv, ok, 0, *sizes)
    assert bwd(at16, at16, at16, at16) == -5
    for i in range(4):
        assert bwd(*[odd if j == i else ok for j in range(4)]) == -9


def test_step_clusters_are_no_larger_than_the_device_places(pkg):
    """Clusters of 16 CTAs are not placed by every device: the launch asks, and takes 8 where they are not."""
    from hattention_b200 import _lib
    f = _lib.lib().llattn_testing_window_step_ranks
    f.argtypes = [ctypes.c_long] + [ctypes.c_int] * 3
    assert f(8, 4100, 4, 16) == 16 and f(8, 4100, 4, 8) == 8 and f(8, 4100, 12, 8) == 8
    for units in (1, 9, 40, 147, 148, 10 ** 9):
        for slots in (1, 256, 257, 5000, 2 ** 30):
            for heads in (1, 8, 9):
                n = f(units, slots, heads, 16)
                assert 1 <= n <= 16 and f(units, slots, heads, 8) == min(n, 8) and (n == 1 or units * n < 2 * 148)
    body = open(os.path.join(CSRC, "window_step.cu")).read()
    body = body[body.index("launch_step("):]
    assert "cudaOccupancyMaxActiveClusters" in body[:body.index("cudaLaunchKernelEx")]
