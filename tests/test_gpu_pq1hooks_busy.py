"""The first use of the Bonsai host hooks while the default stream is busy:
their caches, tables and norms are filled there and read on a stream that does
not wait for it, so the fills have to be done before the hook goes on."""
import test_gpu_pq1hooks as hooks
import pytest

pytestmark = pytest.mark.gpu


class _Busy:
    """a hook whose calls find 20 ms of work queued on the default stream"""

    def __init__(self, fn, torch):
        object.__setattr__(self, "fn", fn)
        object.__setattr__(self, "torch", torch)

    def __setattr__(self, name, value):       # argtypes, restype
        setattr(self.fn, name, value)

    def __call__(self, *args):
        self.torch.cuda._sleep(40_000_000)
        return self.fn(*args)


@pytest.mark.parametrize("kvtq", [0, 4])
def test_layer_hooks_default_stream_busy(oracle, pb, cuda, monkeypatch, kvtq):
    L = pb.lib()
    for name in ("pq1_attn_kv_put", "pq1_attn_fused", "pq1_ffn_fused", "pq1_token_fused"):
        monkeypatch.setattr(L, name, _Busy(getattr(L, name), cuda), raising=False)
    hooks.test_pq1_layer_hooks(oracle, pb, cuda, monkeypatch, kvtq)
