"""The paged K/V cache without a GPU: every entry point refuses what it does
not take before it touches a device (the pointers below are never read), the
scratch sizes, and the 64-bit oracle's own masks, bad pages and eviction
order."""
import ctypes as C

import numpy as np
import pytest

import kv_oracle as KO

P = 0x7F0000000000      # a 16-byte aligned address nothing reads


def pool(pb, **over):
    d = dict(k=P, v=P + (1 << 32), weight=P + (1 << 34), dtype=pb.PB_DT_F16, n_pages=100, page_size=32, n_kv=8,
             head_dim=128, page_stride=8 * 32 * 128, head_stride=32 * 128, row_stride=128)
    d.update(over)
    return pb._KVPages(**d)


class Append(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in "table x seq slot pos qn kn cos sin q".split()] + \
               [(n, C.c_longlong) for n in ("ldx", "ldq")] + \
               [(n, C.c_int) for n in "n_seq table_ld x_dtype n_tok nh half n_rope".split()] + [("eps", C.c_float)]


class Attend(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in "table start len q out scratch".split()] + \
               [(n, C.c_longlong) for n in ("ldq", "ldo", "bytes")] + \
               [(n, C.c_int) for n in "n_seq table_ld max_len nh window sinks od n_tok acc".split()] + [("scale", C.c_float)]


class Evict(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in "table len dst new scratch".split()] + [("bytes", C.c_longlong)] + \
               [(n, C.c_int) for n in "n_seq table_ld max_len dst_ld budget sinks recent".split()]


def call(pb, fn, kind, base, c, over):
    c = pool(pb) if c is None else c
    a = kind(**{**base, **over})
    return getattr(pb.lib(), fn)(C.byref(c), C.cast(C.byref(a), C.c_char_p), None)


def append(pb, c=None, **over):
    return call(pb, "pb_kv_append", Append,
                dict(n_seq=4, table=P, table_ld=10, x=P + (1 << 36), x_dtype=pb.PB_DT_BF16, ldx=48 * 128, n_tok=7, nh=32, seq=P,
                     slot=P, pos=P, qn=P, kn=P, eps=1e-5, cos=P, sin=P, half=64, n_rope=1000, q=P + (1 << 38), ldq=32 * 128), c, over)


ATTEND = dict(n_seq=4, table=P, table_ld=10, len=P, max_len=0, nh=32, q=P + (1 << 36), ldq=32 * 128, scale=0.1, window=0,
              sinks=0, out=P + (1 << 38), od=0, ldo=32 * 128, scratch=P, bytes=1 << 40)


def decode(pb, c=None, **over):
    return call(pb, "pb_kv_decode", Attend, ATTEND, c, over)


def prefill(pb, c=None, **over):
    return call(pb, "pb_kv_prefill", Attend, dict(ATTEND, start=P, n_tok=9), c, over)


def evict(pb, c=None, **over):
    return call(pb, "pb_kv_evict", Evict,
                dict(n_seq=4, table=P, table_ld=10, len=P, max_len=0, dst=P + 4096, dst_ld=8, new=P, budget=200, sinks=4, recent=50,
                     scratch=P, bytes=1 << 40), c, over)


EINVAL, ENOTSUP = -1, -8
BAD_POOLS = [
    (dict(k=None), EINVAL), (dict(v=None), EINVAL), (dict(dtype=1), ENOTSUP), (dict(dtype=7), ENOTSUP),
    (dict(head_dim=96), ENOTSUP), (dict(head_dim=256), ENOTSUP), (dict(page_size=8), ENOTSUP), (dict(page_size=48), ENOTSUP),
    (dict(page_size=512), ENOTSUP), (dict(page_size=0), ENOTSUP), (dict(n_pages=0), EINVAL), (dict(n_kv=0), EINVAL),
    (dict(k=P + 8), EINVAL), (dict(v=P + 2), EINVAL), (dict(row_stride=132), EINVAL), (dict(page_stride=-32768), EINVAL),
    (dict(row_stride=64), EINVAL),            # rows overlap
    (dict(head_stride=31 * 128), EINVAL),     # a head's rows run into the next head's
    (dict(page_stride=0), EINVAL),            # an expanded pool
    (dict(page_stride=1 << 60), EINVAL),      # past 64-bit addresses
]


@pytest.mark.parametrize("call", [append, decode, prefill, evict])
@pytest.mark.parametrize("over,rc", BAD_POOLS)
def test_bad_pools_are_refused(pb, call, over, rc):
    assert call(pb, pool(pb, **over)) == rc
    assert pb.last_error().startswith("pb_kv_")


@pytest.mark.parametrize("call", [append, decode, prefill, evict])
@pytest.mark.parametrize("over", [dict(table=None), dict(table_ld=0), dict(table_ld=1 << 28), dict(n_seq=-1)])
def test_bad_tables_are_refused(pb, call, over):
    assert call(pb, **over) == EINVAL


@pytest.mark.parametrize("over", [
    dict(x=None), dict(seq=None), dict(slot=None), dict(q=None), dict(x_dtype=3), dict(n_tok=-1), dict(nh=0), dict(half=-1),
    dict(half=65), dict(cos=None), dict(sin=None), dict(n_rope=0), dict(ldx=48 * 128 - 8), dict(ldq=31 * 128), dict(x=P + 1),
    dict(q=P + 2), dict(q=P + 8), dict(ldq=32 * 128 + 4), dict(ldq=32 * 128 + 1),
    dict(q=P + (1 << 36) + 16),               # q inside qkv
])
def test_append_refusals(pb, over):
    assert append(pb, **over) == EINVAL


def test_append_of_nothing(pb):
    assert append(pb, n_tok=0) == 0


@pytest.mark.parametrize("call", [decode, prefill])
@pytest.mark.parametrize("over,rc", [
    (dict(len=None), EINVAL), (dict(q=None), EINVAL), (dict(out=None), EINVAL), (dict(od=1), ENOTSUP), (dict(nh=20), ENOTSUP),
    (dict(nh=0), ENOTSUP), (dict(nh=136, ldq=136 * 128, ldo=136 * 128), ENOTSUP), (dict(window=-1), EINVAL),
    (dict(sinks=-1), EINVAL), (dict(scale=0.0), EINVAL), (dict(scale=-1.0), EINVAL), (dict(scale=float("nan")), EINVAL),
    (dict(scale=float("inf")), EINVAL), (dict(ldq=31 * 128), EINVAL), (dict(ldo=31 * 128), EINVAL), (dict(q=P + 8), EINVAL),
    (dict(out=P + 4), EINVAL), (dict(ldo=32 * 128 + 4), EINVAL), (dict(out=P + (1 << 36)), EINVAL),
])
def test_attention_refusals(pb, call, over, rc):
    assert call(pb, **over) == rc


def test_scratch_is_checked(pb):
    L = pb.lib()
    c = pool(pb)
    need = L.pb_kv_decode_scratch(C.byref(c), 4, 320, 32, 1)
    assert need > 0
    assert decode(pb, acc=1, bytes=need - 1) == EINVAL and decode(pb, acc=1, scratch=None) == EINVAL
    assert "scratch" in pb.last_error()
    need = L.pb_kv_evict_scratch(C.byref(c), 4, 320, 200)
    assert need == 4 * 8 * 200 * 4 and L.pb_kv_evict_scratch(C.byref(c), 4, 200, 200) == 0
    assert evict(pb, bytes=need - 1) == EINVAL and evict(pb, scratch=None) == EINVAL
    assert L.pb_kv_decode_scratch(C.byref(c), -1, 320, 32, 1) == -1


def test_weights_are_needed(pb):
    assert decode(pb, pool(pb, weight=None), acc=1) == EINVAL
    assert evict(pb, pool(pb, weight=None)) == EINVAL


@pytest.mark.parametrize("over", [dict(len=None), dict(dst=None), dict(new=None), dict(dst=P), dict(budget=0), dict(sinks=-1),
                                  dict(recent=-1), dict(sinks=151), dict(sinks=201, recent=0), dict(dst_ld=6), dict(dst_ld=0)])
def test_evict_refusals(pb, over):
    assert evict(pb, **over) == EINVAL


@pytest.mark.parametrize("over", [dict(new=P + 4), dict(new=P - 12), dict(scratch=P + 4)])
def test_evict_lengths_in_place_or_apart(pb, over):
    """new_len beside len but sharing entries with it, which the kernels would read after they are replaced; a scratch
    that is not aligned"""
    assert evict(pb, **over) == EINVAL


def test_null_arguments(pb):
    L = pb.lib()
    for fn in (L.pb_kv_append, L.pb_kv_decode, L.pb_kv_prefill, L.pb_kv_evict):
        assert fn(C.byref(pool(pb)), None, None) == EINVAL and fn(None, b"\0" * 256, None) == EINVAL
    assert prefill(pb, start=None) == EINVAL


def test_empty_calls_need_no_pointers(pb):
    """empty torch tensors have null addresses"""
    nothing = dict(table=None, table_ld=0, n_seq=0)
    assert append(pb, n_tok=0, x=None, seq=None, slot=None, q=None) == 0
    assert append(pb, n_tok=0, x=None, seq=None, slot=None, q=None, **nothing) == 0
    assert decode(pb, len=None, q=None, out=None, scratch=None, bytes=0, **nothing) == 0
    assert prefill(pb, n_tok=0, start=None, len=None, q=None, out=None, scratch=None, bytes=0, **nothing) == 0
    assert prefill(pb, n_tok=0, q=None, out=None) == 0
    assert evict(pb, len=None, dst=None, new=None, scratch=None, bytes=0, **nothing) == 0
    assert prefill(pb, n_tok=-1) == EINVAL


def test_packed_arguments_match_the_structs(pb):
    for fmt, kind in ((pb.KVPages._APPEND, Append), (pb.KVPages._ATTEND, Attend), (pb.KVPages._EVICT, Evict)):
        vals = [float(i) if t is C.c_float else i for i, (_, t) in enumerate(kind._fields_, 1)]
        s = kind.from_buffer_copy(fmt.pack(*vals).ljust(C.sizeof(kind), b"\0"))
        assert [getattr(s, n) for n, _ in kind._fields_] == vals


def test_calls_of_no_sequence(pb):
    assert decode(pb, n_seq=0) == 0 and prefill(pb, n_seq=0) == 0 and prefill(pb, n_tok=0) == 0 and evict(pb, n_seq=0) == 0


def test_python_checks_need_cuda_tensors(pb):
    import torch
    with pytest.raises(pb.PBError):
        pb.KVPages(torch.zeros(4, 2, 16, 64, dtype=torch.float16), torch.zeros(4, 2, 16, 64, dtype=torch.float16))


# ------------------------------------------------------------- the oracle
def test_oracle_masks():
    assert KO.seen(5, 9, 0, 0).tolist() == [True] * 6 + [False] * 3
    assert KO.seen(5, 9, 2, 1).tolist() == [True, False, False, False, True, True, False, False, False]
    assert KO.seen(5, 9, 100, 3).tolist() == [True] * 6 + [False] * 3
    assert not KO.seen(-1, 9, 0, 0).any()


def test_oracle_bad_pages_hide_their_rows():
    """rows behind a table entry outside the pool change nothing, whatever it is; the rest is the attention without them"""
    rng = np.random.default_rng(1)
    k, v = rng.standard_normal((5, 1, 16, 64)), rng.standard_normal((5, 1, 16, 64))
    q = rng.standard_normal((2, 64))
    want = KO.attend(q, k, v, None, np.array([[3, 1]]), 0, 31, 32, 0.1, 0, 0)
    for bad in (-1, 5, 2**31 - 1, -2**31):
        got = KO.attend(q, k, v, None, np.array([[3, bad, 1]]), 0, 47, 48, 0.1, 0, 0)
        assert np.allclose(got[0], want[0], rtol=1e-13, atol=0)
        assert (got[4][:, 16:32] == 0).all()
    empty = KO.attend(q, k, v, None, np.array([[-1, 9]]), 0, 31, 32, 0.1, 0, 0)
    assert (empty[0] == 0).all()


def test_oracle_evict_order():
    w = [0, 5, 1, 5, 9, 2, 5, 0]
    assert KO.evict_rows(w, 8, 8, 1, 1) == list(range(8))
    assert KO.evict_rows(w, 8, 4, 1, 1) == [0, 1, 4, 7]           # of the equal fives the lowest row
    assert KO.evict_rows(w, 8, 5, 0, 0) == [1, 3, 4, 5, 6]
    assert KO.evict_rows(w, 8, 2, 1, 1) == [0, 7]
    assert KO.evict_rows([float("nan"), -3, 1, 0], 4, 2, 0, 0) == [0, 2]


def test_oracle_evict_order_with_rows_on_no_page():
    w, all_, n = [0, 5, 1, 5, 9, 2, 5, 0], [True] * 8, 8
    for budget, sinks, recent in ((8, 1, 1), (4, 1, 1), (5, 0, 0), (2, 1, 1)):
        assert KO.evict_rows_named(w, all_, n, budget, sinks, recent) == KO.evict_rows(w, n, budget, sinks, recent)
    some = [False, True, True, False, True, True, True, True]
    assert KO.evict_rows_named(w, some, n, 8, 1, 1) == [1, 2, 4, 5, 6, 7]      # within the budget: moved together
    assert KO.evict_rows_named(w, some, n, 6, 1, 1) == [1, 2, 4, 5, 6, 7]
    assert KO.evict_rows_named(w, some, n, 3, 1, 1) == [1, 4, 7]               # row 0 is not there to stay
    assert KO.evict_rows_named(w, some, n, 4, 0, 3) == [4, 5, 6, 7]
    assert KO.evict_rows_named(w, [False] * 8, n, 3, 1, 1) == []


def test_scratch_sizes_need_the_bound(pb):
    """0 is no bound of rows there (a call takes it as the table's rows, which these functions do not know): the size of
    nothing would be refused by the call behind it"""
    L, c = pb.lib(), C.byref(pool(pb))
    sizes = (lambda s, m: L.pb_kv_decode_scratch(c, s, m, 32, 1), lambda s, m: L.pb_kv_decode_scratch(c, s, m, 32, 0),
             lambda s, m: L.pb_kv_prefill_scratch(c, s, m, 9, 32), lambda s, m: L.pb_kv_evict_scratch(c, s, m, 200))
    for size in sizes:
        assert size(4, 0) == -1 and size(4, -1) == -1 and size(0, -5) == -1
        assert size(0, 0) == 0
        assert size(4, 320) >= 0
    assert decode(pb, acc=1, bytes=sizes[0](4, 320) - 1) == EINVAL      # what max_len 0 stands for
    assert evict(pb, bytes=sizes[3](4, 320) - 1) == EINVAL


def test_python_keeps_few_scratch_sizes(pb):
    """one entry per call shape, of which a server of ragged prompts has no end"""
    h = object.__new__(pb.KVPages)          # (a real one needs CUDA tensors)
    h._need, h._r = {}, C.byref(pool(pb))
    fn = pb.lib().pb_kv_prefill_scratch
    for n in range(5000):
        assert h._bytes(fn, 4, 320, 1 + n % 3000, 32) == fn(h._r, 4, 320, 1 + n % 3000, 32)
    assert len(h._need) <= 1024
