"""GPU tests of the 4-bit operators' bounded waits: when they begin, and what a caller learns of one that runs out.  No fault
is involved: fbmoe_test_expire_grid_wait shortens the limits (2 ms), and set to 1 it also makes waits for one arrival that
never comes."""
import os
import sys

import pytest
import torch

from conftest import REPO

sys.path.insert(0, os.path.join(REPO, "tests"))
from test_gpu_w4 import BF16, Case, check_linear, random_packed  # noqa: E402, F401

pytestmark = pytest.mark.gpu


@pytest.fixture
def expire(fbmoe_lib):
    lib = fbmoe_lib.load_library()

    def set_(mode):
        assert lib.fbmoe_test_expire_grid_wait(mode) == 0
    yield set_
    set_(0)


def long_call(fbmoe_lib):
    """A call of one CTA that lets its successor start at once and takes longer than the shortened limit, and a function
    that makes it."""
    K = 1 << 23
    x = torch.zeros((8, K), dtype=BF16, device="cuda")
    p = torch.zeros((1, K // 128, 1056), dtype=torch.uint8, device="cuda")
    return lambda: fbmoe_lib.linear_w4(x, p)


@pytest.mark.parametrize("T,N,K", [(16, 130, 12288), (64, 18432, 1024)])  # clusters, single CTAs
def test_waits_begin_when_the_predecessor_has_ended(fbmoe_lib, expire, T, N, K):
    p, v = random_packed(N, K, 64, 3)
    x = torch.randn((T, K), generator=torch.Generator().manual_seed(4)).to(BF16).cuda()
    before = long_call(fbmoe_lib)
    before()
    check_linear(fbmoe_lib.linear_w4(x, p, N), x, v, 64)
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    before()
    b.record()
    torch.cuda.synchronize()
    assert a.elapsed_time(b) > 4.0  # twice the limit
    expire(2)
    before()
    y = fbmoe_lib.linear_w4(x, p, N)
    torch.cuda.synchronize()
    check_linear(y, x, v, 64)


@pytest.mark.parametrize("in_place", [False, True])
def test_outputs_of_a_failed_layer_are_nan(fbmoe_lib, expire, in_place):
    """Nothing of what stood in the output, or of what the call got to, is left as if it were a result."""
    c = Case(fbmoe_lib, 9, 32, 0, 256, 128, 64, 64, BF16, "group", 5)
    want = fbmoe_lib.forward_w4(*c.args())
    args = list(c.args())
    args[2] = c.x.clone()
    out = args[2] if in_place else torch.full_like(want, 5.0)
    expire(1)
    with pytest.raises(fbmoe_lib.DeviceStatusError):
        fbmoe_lib.forward_w4(*args, out=out, sync_status=True)
    expire(0)
    assert out.isnan().all()
    assert torch.equal(fbmoe_lib.forward_w4(*c.args(), sync_status=True), want)


def test_a_failed_call_is_reported_once_and_by_itself(fbmoe_lib, expire):
    """A call that fails on one stream, and one that succeeds after it on another and asks for its own status."""
    c = Case(fbmoe_lib, 5, 32, 0, 256, 128, 64, 64, BF16, "group", 6)
    want = fbmoe_lib.forward_w4(*c.args(), sync_status=True)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    expire(1)
    with torch.cuda.stream(a):
        fbmoe_lib.forward_w4(*c.args())     # fails 2 ms from now
    expire(0)
    told = 0
    with torch.cuda.stream(b):
        try:
            y = fbmoe_lib.forward_w4(*c.args(), sync_status=True)  # its own status is clean
        except fbmoe_lib.DeviceStatusError as e:  # this thread was held up until the first call had failed
            assert "earlier" in str(e)
            told, y = 1, fbmoe_lib.forward_w4(*c.args(), sync_status=True)
    assert torch.equal(y, want)
    try:
        fbmoe_lib.check_status()
    except fbmoe_lib.DeviceStatusError:
        told += 1
    assert told >= 1  # twice, if the first report came while its CTAs were still giving up
    fbmoe_lib.check_status()
    expire(1)
    with pytest.raises(fbmoe_lib.DeviceStatusError):
        fbmoe_lib.forward_w4(*c.args(), sync_status=True)
    expire(0)
    fbmoe_lib.check_status()                # it has been reported


def test_two_threads_get_their_own_status(fbmoe_lib, expire):
    """Two threads whose calls all fail, each asking for its own status: none takes the other's."""
    import threading
    cases = [Case(fbmoe_lib, T, 16, 0, 256, 128, 64, 64, BF16, "group", T) for T in (3, 7)]
    for c in cases:
        fbmoe_lib.forward_w4(*c.args(), sync_status=True)
    torch.cuda.synchronize()
    seen = [[], []]

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(12):
                try:
                    fbmoe_lib.forward_w4(*cases[k].args(), sync_status=True)
                    seen[k].append("none")
                except fbmoe_lib.DeviceStatusError as e:
                    seen[k].append("own" if "this forward_w4" in str(e) else "other")

    expire(1)
    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    expire(0)
    torch.cuda.synchronize()
    assert seen == [["own"] * 12] * 2
    fbmoe_lib.check_status()


def test_a_graph_captured_before_the_first_call_reports_its_status():
    """In a process whose first 4-bit call on the device is a captured one."""
    import subprocess
    code = r"""
import os, sys
sys.path[:0] = [os.path.join(os.environ["FBMOE_REPO"], "flashinfer-bench-moe_b200"), os.path.join(os.environ["FBMOE_REPO"], "tests")]
import torch
import fbmoe_lib as L
from test_gpu_w4 import Case, BF16, random_packed
c = Case(L, 4, 32, 0, 256, 128, 64, 64, BF16, "group", 7)
graphs, outs = [], []
for mode in (1, 0):
    L.load_library().fbmoe_test_expire_grid_wait(mode)
    graphs.append(torch.cuda.CUDAGraph())
    with torch.cuda.graph(graphs[-1]):
        outs.append(L.forward_w4(*c.args()))
graphs[1].replay()
L.check_status()
c.check(outs[1])
graphs[0].replay()
try:
    L.check_status()
    print("silent")
except L.DeviceStatusError as e:
    print("word", e.word)
graphs[1].replay()
L.check_status()
c.check(outs[1])
"""
    r = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, FBMOE_REPO=REPO), capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-3000:]
    assert r.stdout.split() == ["word", "4"]


@pytest.mark.parametrize("T,N,K", [(16, 130, 12288), (64, 18432, 1024)])  # clusters, single CTAs
def test_a_failed_linear_is_nan_and_reported(fbmoe_lib, expire, T, N, K):
    p, v = random_packed(N, K, 64, 3)
    x = torch.randn((T, K), generator=torch.Generator().manual_seed(4)).to(BF16).cuda()
    want = fbmoe_lib.linear_w4(x, p, N)
    expire(1)
    out = torch.full((T + 1, N + 8), 7.0, dtype=BF16, device="cuda")
    fbmoe_lib.linear_w4(x, p, N, out=out[:T, 4:N + 4])
    expire(0)
    with pytest.raises(fbmoe_lib.DeviceStatusError) as e:
        fbmoe_lib.check_status()
    assert e.value.word & 4
    assert out[:T, 4:N + 4].isnan().all()
    assert (out[:, :4] == 7).all() and (out[:, N + 4:] == 7).all() and (out[T] == 7).all()
    assert torch.equal(fbmoe_lib.linear_w4(x, p, N), want)
    fbmoe_lib.check_status()
    expire(1)
    fbmoe_lib.linear_w4(x, p, N)
    expire(0)
    torch.cuda.synchronize()
    with pytest.raises(fbmoe_lib.DeviceStatusError):
        fbmoe_lib.linear_w4(x, p, N)        # the next call says so
    assert torch.equal(fbmoe_lib.linear_w4(x, p, N), want)
    fbmoe_lib.check_status()


def test_a_captured_linear_reports_its_status(fbmoe_lib, expire):
    p, _ = random_packed(130, 12288, 64, 3)
    x = torch.randn((12, 12288), generator=torch.Generator().manual_seed(4)).to(BF16).cuda()
    want = fbmoe_lib.linear_w4(x, p, 130)
    expire(1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = fbmoe_lib.linear_w4(x, p, 130)
    expire(0)
    for _ in range(2):
        graph.replay()
        with pytest.raises(fbmoe_lib.DeviceStatusError):
            fbmoe_lib.check_status()
        assert y.isnan().all()
    assert torch.equal(fbmoe_lib.linear_w4(x, p, 130), want)
