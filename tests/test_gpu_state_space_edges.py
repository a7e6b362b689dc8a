"""State-space operators and the 4-bit product where they can go wrong: busy memory,
accuracy, decays, non-finite values, calls from several threads and streams, limits."""
import pytest
import torch

from cpp1_b200 import ops
from test_gpu_state_space import gen, i32, make_scan, offs, rnd, scan_ref, scan_tol, state_tol, within

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


@pytest.mark.parametrize("lens,h,n", [([128] * 24, 64, 128), ([256] * 9, 40, 128), ([300, 90, 513], 148, 64)])
def test_scan_beside_busy_memory(cuda, lens, h, n):
    """The tensor-core scan's loads arrive in any order when other streams keep the memory
    busy: chunks whose C lands long after B and x give the same bits as on a quiet GPU."""
    b = offs(lens)
    a = make_scan(h, b[-1], h, 64, 1, n, "bf16")
    st = rnd(gen(h), len(lens), h, 64, n)
    ref, mag, (fin, fmag) = scan_ref(a, b, st)
    so = torch.empty_like(st)
    o = i32(b)
    y = ops.selective_scan(**a, offsets=o, state=st, state_out=so)
    within(y, ref, scan_tol(ref, mag, n, max(lens), BF, True), "y")
    within(so, fin, state_tol(fin, fmag, max(lens), True), "state")
    big = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    other = torch.empty_like(big)
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(15):
        for s in side:
            with torch.cuda.stream(s):
                other.copy_(big)
        so2 = torch.empty_like(st)
        y2 = ops.selective_scan(**a, offsets=o, state=st, state_out=so2)
        torch.cuda.synchronize()
        assert torch.equal(y2, y) and torch.equal(so2, so)
