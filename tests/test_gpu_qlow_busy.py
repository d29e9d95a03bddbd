"""A Q4 matrix packed on a stream of its own while the default stream is busy:
its error word is cleared before the pack returns, not behind what is queued
on the default stream, where the clearing would take a report away."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


class _Head(C.Structure):
    """the library's handle: bits, N, K, codes, scales, error word"""
    _fields_ = [("bits", C.c_int), ("N", C.c_int), ("K", C.c_int), ("codes", C.c_void_p), ("scales", C.c_void_p),
                ("err", C.c_void_p)]


def test_pack_while_the_default_stream_is_busy(oracle, pb, cuda):
    torch = cuda
    from pulsar_b200 import synth
    N, K = 96, 4096
    codes, scales = synth.qlow_payload(np.random.default_rng(3), N, K, 4)
    x = np.random.default_rng(4).integers(0x3F00, 0x4000, K).astype(np.uint16)
    xd = torch.from_numpy(x.view(np.int16)).cuda()
    y = torch.empty(N, dtype=torch.int16, device="cuda")
    side, keep = torch.cuda.Stream(), []
    for cycles in (1000, 2_000_000_000):     # the first time modules are loaded, which waits for the device; then about 1 s
        torch.cuda.synchronize()
        torch.cuda._sleep(cycles)
        w = pb.QlowTensor(codes, scales, 4, N, K, stream=side)
        keep.append(w)                        # (freeing it waits for the device)
        w.gemv(xd, y, stream=side)
        head = _Head.from_address(w.h.value)
        assert (head.bits, head.N, head.K) == (4, N, K)

        class Word:
            __cuda_array_interface__ = dict(data=(head.err, False), shape=(1,), typestr="<i4", version=3)

        with torch.cuda.stream(side):
            word = torch.as_tensor(Word(), device="cuda")
            word.fill_(1)                     # as a product that gave up does
        side.synchronize()
        busy = not torch.cuda.default_stream().query()
        with pytest.raises(pb.PBError, match="gave up"):
            w.status(side)
    assert busy, "the default stream was not busy: no test"
    word.zero_()
    torch.cuda.synchronize()
    w.status()
    assert np.array_equal(y.cpu().numpy().view(np.uint16), oracle.qlow_gemv(codes, scales, 4, N, K, x))
