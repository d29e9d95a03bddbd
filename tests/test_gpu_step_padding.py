"""A model narrower than the GEMV's 2048-code segments: the weights' rows are
padded with zero codes, so the padding of the input vector in shared memory
must be finite too (0 times a NaN left there by an earlier kernel is NaN). An
attention over cache rows of all one bits first leaves NaN patterns in every
SM's shared memory."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_narrow_model_after_nan_shared_memory(tmp_path, oracle, pb, cuda):
    torch = cuda
    from pulsar_b200 import synth
    c = dict(synth.LFM3_TINY, hidden=256, inter=512, n_heads=4, n_kv=2, head_dim=64, vocab=512, n_layers=2, attn_layers=(1,))
    w = synth.make_weights(c, seed=8)
    path = str(tmp_path / "narrow.lfm3q8")
    synth.write_model(path, c, w)
    ones = torch.full((600, 8, 64, 64), -1, dtype=torch.int16, device="cuda").view(torch.float16)
    cache = pb.KVPages(ones, ones.clone())
    table = torch.arange(600, dtype=torch.int32, device="cuda").view(1, 600)
    length = torch.tensor([600 * 64], dtype=torch.int32, device="cuda")
    q = torch.zeros((1, 32, 64), dtype=torch.float16, device="cuda")
    out = torch.empty_like(q)
    m = pb.Model(path)
    s = m.new_state(16)
    om = oracle.Model(synth.oracle_cfg(c, 16), w)
    logits = torch.empty(c["vocab"], dtype=torch.float32, device="cuda")
    tok = 7
    for pos in range(6):
        cache.decode(table, length, q, out)
        torch.cuda.synchronize()
        got = s.decode_token(tok, pos, logits=logits)
        want, lg, _ = om.decode(tok, pos, want_logits=True)
        torch.cuda.synchronize()
        assert np.array_equal(logits.cpu().numpy().view(np.uint32), lg.view(np.uint32)), "pos %d" % pos
        assert got == want
        tok = got
    s.destroy()
    m.close()
