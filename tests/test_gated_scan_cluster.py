"""The gated scan over clusters of blocks: every form of it against the 64-bit oracle with a clean status word, and what
happens when the maps of a step do not come."""
import time

import pytest
import torch

from oracle import recurrent_oracle as orc
from triton_snn_fusion_b200 import _lib
from triton_snn_fusion_b200.runtime import temporal_gated_scan_backend as ops

DEV = "cuda"
pytestmark = pytest.mark.gpu


def _inputs(T, B, D, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x, dh = (torch.randn(B, T, D, generator=g).to(dtype) for _ in range(2))
    gate = (torch.randn(B, T, D, generator=g) * 1.5 + 2).clamp(-8, 8).to(dtype)
    return x, gate, torch.randn(B, D, generator=g) * 0.5, dh, torch.randn(B, D, generator=g)


def _both(x, gate, h0, dh, dl, lengths=None):
    kw = dict(batch_first=True, lengths=lengths)
    f = ops.run_temporal_gated_scan(x, gate, h0, save_for_backward=True, **kw)
    return f, ops.run_temporal_gated_scan_backward(dh, x, gate, h0, f.ckpt, dh_last=dl, **kw)


def _against_oracle(cpu, f, r, lengths=None):
    x, gate, h0, dh, dl = cpu
    t = lambda v: v.transpose(0, 1)  # noqa: E731
    h, eh, last, el = orc.gated_scan(t(x), t(gate), h0, "sigmoid", True, lengths)
    orc.assert_within(t(f.h_seq), h, eh, "h_seq")
    orc.assert_within(f.h_last, last, el, "h_last")
    ref, err = orc.gated_scan_backward(t(dh), dl, t(x), t(gate), h0, "sigmoid", True, lengths)
    for name, got, want, e in zip(("dx", "dgate", "dh_init"), (t(r.dx), t(r.dgate), r.dh_init), ref, err):
        orc.assert_within(got, want, e, name)


# two, four and eight blocks a sequence and fewer tiles of time than that; rows on 16-byte boundaries and others
@pytest.mark.parametrize("T,B,D", [(200, 1, 64), (400, 2, 96), (1100, 1, 64), (3000, 1, 32), (520, 4, 2048), (700, 2, 1024),
                                   (1100, 1, 65), (900, 3, 33), (2100, 1, 1023)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_clusters_leave_a_clean_status(T, B, D, dtype):
    assert _lib.device_status() == 0
    cpu = _inputs(T, B, D, dtype, seed=T)
    dev = [t.to(DEV) for t in cpu]
    _against_oracle(cpu, *_both(*dev))
    if B > 1:
        n = torch.tensor([0, T, T // 2 + 1, 1][:B], dtype=torch.int32)
        _against_oracle(cpu, *_both(*dev, n.to(DEV)), n)
    assert _lib.device_status() == 0


@pytest.mark.parametrize("D", [64, 65])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("backward", [False, True])
def test_a_map_that_does_not_come_ends_in_a_status(D, dtype, backward):
    """The last block of the first cluster waits in the first step for a map that nobody sends, the limit of the waits being
    about a millisecond. That block gives up in the first step, the others of its cluster in the second, where its maps are missing;
    the call ends by itself, the status word says so once, and the next call is right again."""
    T, B = 2500, 2
    cpu = _inputs(T, B, D, dtype)
    dev = [t.to(DEV) for t in cpu]
    f, r = _both(*dev)
    assert _lib.device_status() == 0
    _lib.check(_lib.lib.snnb_selftest_arm_wait_timeout(2_000_000), "arm")
    t0 = time.perf_counter()
    if backward:
        ops.run_temporal_gated_scan_backward(dev[3], *dev[:3], f.ckpt, dh_last=dev[4], batch_first=True)
    else:
        ops.run_temporal_gated_scan(*dev[:3], batch_first=True)
    torch.cuda.synchronize()
    assert time.perf_counter() - t0 < 1.0
    assert _lib.device_status() != 0
    assert _lib.device_status() == 0
    again = _both(*dev)
    for p, q in zip((*f, *r), (*again[0], *again[1])):
        assert torch.equal(p, q)
    _against_oracle(cpu, *again)
    assert _lib.device_status() == 0
