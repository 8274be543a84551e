"""CPU: refusals of the paged-cache operators before anything is launched, and their size queries. The C entries return
an error for every argument that their kernels could not address; the Python functions raise."""
import ctypes
import math
from pathlib import Path

import pytest
import torch

import paged_oracle as oracle

LIB = Path(__file__).resolve().parents[1] / "qwentts-turbo_amd" / "lib" / "libqwentts_amd.so"
P, I, L, F, Z = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_float, ctypes.c_size_t
INVALID = 1                       # hipErrorInvalidValue
A = 1 << 20                       # an aligned address that nothing reads

class Cache(ctypes.Structure):
    _fields_ = [("k", P), ("v", P), ("dtype", I), ("num_pages", I), ("page_size", I), ("num_kv_heads", I), ("head_dim", I),
                ("page_stride", L), ("head_stride", L), ("slot_stride", L)]

def cache(**kw):
    d = dict(k=A, v=A, dtype=0, num_pages=4, page_size=16, num_kv_heads=8, head_dim=128, page_stride=8 * 16 * 128,
             head_stride=16 * 128, slot_stride=128)
    d.update(kw)
    return Cache(**d)

@pytest.fixture(scope="module")
def lib():
    if not LIB.exists():
        pytest.skip("libqwentts_amd.so is not built")
    x = ctypes.CDLL(str(LIB))
    x.qtts_paged_plan.argtypes = [I, I, L, I, I, P, P, P, P, I, P] + [P] * 7 + [P]
    x.qtts_paged_release.argtypes = [I, I, L, I, P, P, P, P, I, P, P]
    x.qtts_qk_norm_rope_store.argtypes = [P, I, I, P, L, L, P, L, L, P, L, L, P, L, L, P, P, F, P, P, I, I, P, L, I, I, P, P]
    x.qtts_paged_attention_decode.argtypes = [P, I, I, P, L, L, P, L, L, P, I, L, P, I, F, I, I, P, Z, P]
    x.qtts_paged_attention_prefill.argtypes = [P, I, I, I, P, L, L, P, L, L, P, I, L, P, P, I, F, I, I, P]
    x.qtts_paged_decode_workspace_bytes.argtypes = [I] * 9
    x.qtts_paged_decode_workspace_bytes.restype = Z
    x.qtts_backbone_paged.argtypes = [P, Z, P, P, I, P, P, P, I, P, L, I, I, P, P, P, P, P, I, L, I, I, I, P, P, P, I, P, P, I, P, I, P, I, F,
                                      I, I, P, I, P, P]
    x.qtts_paged_workspace_bytes.argtypes = [I] * 8
    x.qtts_paged_workspace_bytes.restype = Z
    return x

BAD_CACHES = [dict(k=0), dict(v=0), dict(k=A + 8), dict(v=A + 2), dict(dtype=2), dict(dtype=-1), dict(num_pages=0), dict(num_kv_heads=0),
              dict(head_dim=96), dict(head_dim=256), dict(page_size=8), dict(page_size=48), dict(page_size=0), dict(page_size=1 << 17),
              dict(page_stride=1004), dict(page_stride=-8), dict(page_stride=1 << 31), dict(head_stride=4), dict(head_stride=1 << 31),
              dict(slot_stride=64), dict(slot_stride=132), dict(slot_stride=(1 << 24) + 8)]

def store(lib, c=None, **kw):
    d = dict(n=3, hq=16, q=A, qt=2048, qh=128, k=A, kt=1024, kh=128, v=A, vt=1024, vh=128, o=A, ot=2048, oh=128, wq=A, wk=A, eps=1e-6,
             cos=A, sin=A, f32=0, rows=10, pos=A, ps=0, h=0, w=0, slots=A)
    d.update(kw)
    return lib.qtts_qk_norm_rope_store(ctypes.byref(c) if c is not None else None, *d.values(), None)

def decode(lib, c=None, **kw):
    d = dict(n=3, hq=16, q=A, qt=2048, qh=128, o=A, ot=2048, oh=128, table=A, width=4, stride=4, lens=A, max_len=64, scale=0.1, window=0,
             sinks=0, ws=A, wsb=1 << 30)
    d.update(kw)
    return lib.qtts_paged_attention_decode(ctypes.byref(c) if c is not None else None, *d.values(), None)

def prefill(lib, c=None, **kw):
    d = dict(n=3, t=9, hq=16, q=A, qt=2048, qh=128, o=A, ot=2048, oh=128, table=A, width=4, stride=4, lens=A, cu=A, max_len=64, scale=0.1,
             window=0, sinks=0)
    d.update(kw)
    return lib.qtts_paged_attention_prefill(ctypes.byref(c) if c is not None else None, *d.values(), None)

@pytest.mark.parametrize("bad", BAD_CACHES, ids=str)
def test_caches_that_kernels_cannot_address(lib, bad):
    for call in (store, decode, prefill):
        assert call(lib, cache(**bad)) == INVALID, call.__name__

def test_store_refusals(lib):
    c = cache()
    assert store(lib) == INVALID                                            # no cache
    for bad in (dict(n=-1), dict(hq=0), dict(q=0), dict(k=0), dict(v=0), dict(o=0), dict(cos=0), dict(sin=0), dict(pos=0), dict(slots=0),
                dict(q=A + 4), dict(o=A + 8), dict(cos=A + 2), dict(wk=A + 2), dict(qt=2049), dict(qh=130), dict(kt=4), dict(vh=1), dict(oh=12),
                dict(rows=0), dict(ps=-1), dict(h=65), dict(w=-1), dict(eps=-1.0), dict(eps=math.nan)):
        assert store(lib, c, **bad) == INVALID, bad
    assert store(lib, c, n=0) == 0                                          # nothing to do, nothing launched

def test_attention_refusals(lib):
    c = cache()
    assert decode(lib) == INVALID and prefill(lib) == INVALID
    for bad in (dict(n=0), dict(hq=0), dict(hq=12), dict(q=0), dict(o=0), dict(table=0), dict(lens=0), dict(q=A + 2), dict(o=A + 8),
                dict(qt=3), dict(oh=4), dict(width=0), dict(stride=3), dict(width=(1 << 26) + 1, stride=1 << 27), dict(max_len=0), dict(scale=0.0),
                dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan), dict(window=-1), dict(sinks=-1)):
        assert decode(lib, c, **bad) == INVALID, bad
        assert prefill(lib, c, **bad) == INVALID, bad
    assert prefill(lib, c, cu=0) == INVALID and prefill(lib, c, t=-1) == INVALID and prefill(lib, c, t=0) == 0
    # a split call needs its workspace, aligned and large enough
    big = dict(n=1, width=1000, stride=1000, max_len=16000)
    need = lib.qtts_paged_decode_workspace_bytes(1, 16, 8, 128, 1000, 16, 16000, 0, 0)
    assert need > 0
    for bad in (dict(ws=0), dict(wsb=need - 1), dict(ws=A + 8)):
        assert decode(lib, c, **big, **bad) == INVALID, bad

def test_plan_and_release_refusals(lib):
    def plan(**kw):
        d = dict(n=2, width=4, stride=4, page=16, total=8, new=A, len=A, table=A, free=A, cap=9, count=A, slots=A, pos=A, cu=A, kv=A, lo=A,
                 fo=A, st=A)
        d.update(kw)
        return lib.qtts_paged_plan(*d.values(), None)
    for bad in (dict(n=0), dict(width=0), dict(stride=3), dict(page=0), dict(page=24), dict(page=1 << 17), dict(total=-1), dict(cap=-1),
                dict(width=(1 << 14) + 1, stride=1 << 20, page=1 << 16), dict(free=0), dict(total=(1 << 30) + 1), dict(n=(1 << 24) + 1), *(dict([(k, 0)]) for k in
                ("new", "len", "table", "count", "slots", "pos", "cu", "kv", "lo", "fo", "st"))):
        assert plan(**bad) == INVALID, bad

    def release(**kw):
        d = dict(n=2, width=4, stride=4, page=16, rel=A, len=A, table=A, free=A, cap=9, count=A)
        d.update(kw)
        return lib.qtts_paged_release(*d.values(), None)
    for bad in (dict(n=0), dict(width=0), dict(stride=1), dict(page=17), dict(cap=0), *(dict([(k, 0)]) for k in
                ("rel", "len", "table", "free", "count"))):
        assert release(**bad) == INVALID, bad

def test_backbone_refusals(lib):
    need = lib.qtts_paged_workspace_bytes(3, 3, 256, 4, 16, 64, 0, 0)
    assert need > 0

    def run(c, **kw):
        d = dict(ws=A, wsb=need, layers=A, host=A, nl=2, norm=A, cos=A, sin=A, rows=64, cache=ctypes.byref(c) if c is not None else None,
                 ls=0, n=3, t=3, slots=A, pos=A, cu=0, kv=A, table=A, width=4, stride=4, max_len=64, window=0, sinks=0, x=A, hidden=A,
                 head=A, vocab=256, logits=0, tokens=A, mask=0, hist=0, hs=0, nh=0, hl=0, rep=1.0, eos=-1, sup=0, sampling=0, frame=0,
                 skip=0)
        d.update(kw)
        return lib.qtts_backbone_paged(*d.values(), None)
    for bad in BAD_CACHES + [dict(dtype=1), dict(num_kv_heads=4), dict(head_dim=64, slot_stride=64)]:
        assert run(cache(**bad)) == INVALID, bad
    assert run(None) == INVALID
    for bad in (*(dict([(k, 0)]) for k in ("ws", "layers", "host", "nl", "norm", "cos", "sin", "rows", "n", "t", "slots", "pos", "kv", "table",
                                           "width", "max_len", "x", "hidden", "tokens")),
                dict(ws=A + 128), dict(wsb=need - 1), dict(ls=-8), dict(ls=4), dict(t=4), dict(t=(1 << 20) + 1, cu=A), dict(stride=3),
                dict(width=(1 << 26) + 1, stride=1 << 27), dict(window=-1), dict(sinks=-1), dict(x=A + 2), dict(vocab=100), dict(vocab=8192)):
        assert run(cache(), **bad) == INVALID, bad

def test_workspace_queries(lib):
    f, g = lib.qtts_paged_decode_workspace_bytes, lib.qtts_paged_workspace_bytes
    assert f(0, 16, 8, 128, 4, 16, 9, 0, 0) == 0 and f(1, 12, 8, 128, 4, 16, 9, 0, 0) == 0
    assert f(1, 16, 8, 128, 4, 16, 64, 0, 0) == 0                           # short: one unit, no workspace
    one = f(1, 16, 8, 128, 4096, 16, 65536, 0, 0)
    assert one > 0 and one % (16 * 130 * 4) == 0                            # sums of every head and unit, with their max and sum
    assert f(1, 16, 8, 128, 4096, 16, 65536, 100, 4) < one                  # a window bounds the units
    assert g(0, 1, 0, 4, 16, 9, 0, 0) == 0 and g(1, 1, 3073, 4, 16, 9, 0, 0) == 0
    assert 0 < g(1, 1, 0, 4, 16, 9, 0, 0) < g(64, 64, 3072, 4, 16, 9, 0, 0)

def test_python_functions_refuse_host_tensors(pkg):
    z = torch.zeros(4, dtype=torch.int32)
    kv = torch.zeros(4, 8, 16, 128, dtype=torch.bfloat16)
    q = torch.zeros(4, 16, 128, dtype=torch.bfloat16)
    t = torch.zeros(4, 4, dtype=torch.int32)
    tab = torch.zeros(8, 128, dtype=torch.bfloat16)
    for call in (lambda: pkg.paged_plan(z, z, t, z, z[:1], 16, 4), lambda: pkg.paged_release(z, z, t, z, z[:1], 16),
                 lambda: pkg.qk_norm_rope_store(q, q[:, :8], q[:, :8], None, None, tab, tab, z, z, kv, kv),
                 lambda: pkg.paged_attention_decode(q, kv, kv, t, z), lambda: pkg.paged_attention_prefill(q, kv, kv, t, z, z)):
        with pytest.raises(RuntimeError, match="GPU tensor"):
            call()

def test_oracle_plan_by_hand():
    """The plan's oracle on a case worked out by hand: pages of 4, stack [7, 8, 9] with 9 on top."""
    table = [[5, -1, -1], [-1, -1, -1], [6, -1, -1]]
    r = oracle.plan([2, 5, 1], [3, 0, 4], table, [7, 8, 9], 3, 4, 8)
    assert table == [[5, 9, -1], [8, 7, -1], [6, -1, -1]]
    assert r == dict(slots=[23, 36, 32, 33, 34, 35, 28, -1], positions=[3, 4, 0, 1, 2, 3, 4, 4], cu=[0, 2, 7, 8], kv=[5, 5, 0],
                     held=[5, 5, 4], status=[0, 0, 1], count=0)

def test_oracle_attention_against_a_dense_softmax():
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(3, 2, 16, 64, generator=g, dtype=torch.float64) for _ in range(2))
    q = torch.randn(1, 4, 64, generator=g, dtype=torch.float64)
    out, _ = oracle.attend(q, k, v, [[2, 0]], [20], 2, 7, 3, 0.25)
    seen = [0, 1, 2] + list(range(14, 21))
    kk, vv = (torch.cat((x[2], x[0]), 1)[:, seen] for x in (k, v))
    s = torch.einsum("hd,hkd->hk", q[0], kk.repeat_interleave(2, 0)) * 0.25
    ref = torch.einsum("hk,hkd->hd", torch.softmax(s, -1), vv.repeat_interleave(2, 0))
    assert float((out[0] - ref).abs().max()) < 1e-12
