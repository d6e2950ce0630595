"""Arguments that the calls of the 4-bit cache and the beam selection refuse, before anything touches a device (the context is the
last thing they look at, so no GPU is needed), and the sizes that their workspaces report."""
import ctypes

import numpy as np
import pytest

import malkin_amd as mk_
import kv4_cases as cases

X = 1 << 20  # a 16-byte aligned address that nothing reads


def refused(rc, code, text):
    assert rc == code, rc
    assert text in mk_.load().mk_last_error().decode(), mk_.load().mk_last_error()


def cache(**over):
    f = dict(k=X, v=X, k_scale=X, v_scale=X, table=X, len=X, refs=X, n_layer=2, n_page=40, page=32, n_head_kv=2, head_dim=128,
             n_seq=3, max_pages=8)
    f.update(over)
    return mk_.MkKv4Cache(*(f[n] for n, _ in mk_.MkKv4Cache._fields_))


def call(name, order, over, **defaults):
    a = dict(defaults)
    a.update(over)
    args = [ctypes.byref(a[x]) if isinstance(a[x], ctypes.Structure) else a[x] for x in order.split()]
    return getattr(mk_.load(), name)(None, *args)


def tables(**over):
    r = dict(dim=128, scaling=mk_.ROPE_YARN, base=1e6, factor=4.0, n_orig=32768, beta_fast=32.0, beta_slow=1.0, attn_factor=0.0)
    r.update({k: over.pop(k) for k in list(over) if k in r})
    return call("mk_rope_tables", "rope divide first n cos sin", over, rope=mk_.MkRope(*r.values()), divide=None, first=0, n=10,
                cos=X, sin=X)


def rope(**over):
    return call("mk_rope_kv4", "q k v stride n H qn kn eps layout dim cos sin pos rpos seq row kv layer out os", over, q=X, k=X,
                v=X, stride=1024, n=5, H=4, qn=X, kn=X, eps=1e-6, layout=0, dim=128, cos=X, sin=X, pos=100, rpos=X, seq=X, row=X,
                kv=cache(), layer=1, out=X + 64, os=512)


def rows(**over):
    return call("mk_kv4_rows", "kv layer seq row n k v", over, kv=cache(), layer=1, seq=X, row=X, n=5, k=X, v=X)


def attention(**over):
    return call("mk_attention_kv4", "q qs out os n H kv layer seq keys most run xq ws wsb", over, q=X, qs=512, out=X, os=512, n=5,
                H=4, kv=cache(), layer=1, seq=X, keys=X, most=256, run=1, xq=None, ws=X, wsb=1 << 40)


def fork(**over):
    return call("mk_kv4_fork", "kv dst src n ws wsb", over, kv=cache(), dst=None, src=X, n=3, ws=X, wsb=1 << 40)


def resize(**over):
    return call("mk_kv4_resize", "kv seq len n st ws wsb", over, kv=cache(), seq=None, len=X, n=3, st=X, ws=X, wsb=1 << 40)


def compact(**over):
    return call("mk_kv4_compact", "kv live ws wsb", over, kv=cache(), live=X, ws=X, wsb=1 << 40)


def beam(**over):
    return call("mk_beam_select", "l stride groups beams V s done eos k os oq ot ws wsb", over, l=X, stride=1000, groups=2, beams=4,
                V=1000, s=X, done=X, eos=3, k=8, os=X, oq=X, ot=X, ws=X, wsb=1 << 40)


@pytest.mark.parametrize("over,text", [
    (dict(rope=None), "null parameters"), (dict(dim=0), "dim"), (dict(dim=3), "dim"), (dict(dim=258), "dim"),
    (dict(scaling=4), "scaling"), (dict(scaling=-1), "scaling"), (dict(base=0.0), "base"), (dict(base=float("inf")), "base"),
    (dict(base=float("nan")), "base"), (dict(factor=0.0), "factor"), (dict(factor=float("nan")), "factor"),
    (dict(scaling=mk_.ROPE_NTK, dim=2), "more than one pair"), (dict(n_orig=0), "YaRN"), (dict(base=1.0), "YaRN"),
    (dict(beta_fast=0.0), "YaRN"), (dict(beta_slow=-1.0), "YaRN"), (dict(attn_factor=float("inf")), "YaRN"),
    (dict(n=-1), "positions"), (dict(first=-1), "positions"), (dict(first=2 ** 31 - 9), "positions"), (dict(cos=None), "null array"),
    (dict(sin=None), "null array"), (dict(), "null context"), (dict(scaling=0, factor=0.0, n_orig=0), "null context"),
    (dict(first=2 ** 31 - 10), "null context"),
])
def test_tables(over, text):
    refused(tables(**over), mk_.MK_ERR_INVALID, text)


BAD_CACHES = [
    (dict(kv=None), "null cache"), (dict(kv=cache(n_layer=0)), "cache sizes"), (dict(kv=cache(n_page=0)), "cache sizes"),
    (dict(kv=cache(n_head_kv=0)), "cache sizes"), (dict(kv=cache(n_seq=0)), "cache sizes"), (dict(kv=cache(max_pages=0)), "cache sizes"),
    (dict(kv=cache(page=8)), "power of two"), (dict(kv=cache(page=48)), "power of two"), (dict(kv=cache(page=2048)), "power of two"),
    (dict(kv=cache(k=0)), "null cache array"), (dict(kv=cache(v_scale=0)), "null cache array"), (dict(kv=cache(table=0)), "null cache array"),
    (dict(kv=cache(k=X + 8)), "not aligned"), (dict(kv=cache(v=X + 4)), "not aligned"), (dict(kv=cache(k_scale=X + 4)), "not aligned"),
    (dict(kv=cache(v_scale=X + 8)), "not aligned"), (dict(kv=cache(max_pages=1 << 26)), "too large"),
    (dict(kv=cache(n_seq=1 << 28)), "too large"), (dict(kv=cache(n_layer=1 << 19)), "too large"),
    (dict(kv=cache(n_page=1 << 30)), "too large"), (dict(kv=cache(n_page=1 << 27)), "too large"),
]


@pytest.mark.parametrize("over,text", BAD_CACHES)
@pytest.mark.parametrize("f", [rope, rows, attention, fork, resize, compact])
def test_caches(f, over, text):
    refused(f(**over), mk_.MK_ERR_INVALID, text)
    name = {"rope": "mk_rope_kv4", "rows": "mk_kv4_rows", "attention": "mk_attention_kv4"}.get(f.__name__, "mk_kv4_" + f.__name__)
    assert mk_.load().mk_last_error().decode().startswith(name + ": ")


@pytest.mark.parametrize("f", [rope, rows, attention, fork, resize, compact])
def test_head_dims(f):
    for d in (32, 96, 256):
        refused(f(kv=cache(head_dim=d)), mk_.MK_ERR_UNSUPPORTED, "head_dim")


@pytest.mark.parametrize("f", [rope, rows, attention])
def test_layers_and_lengths(f):
    for layer in (-1, 2):
        refused(f(layer=layer), mk_.MK_ERR_INVALID, "bad layer")
    # These read the table alone.
    refused(f(kv=cache(len=0, refs=0)), mk_.MK_ERR_INVALID, "null context")
    refused(f(n=-1), mk_.MK_ERR_INVALID, "bad sizes")
    assert f(n=0, kv=None) == mk_.MK_OK


@pytest.mark.parametrize("f", [fork, resize, compact])
def test_pools(f):
    refused(f(kv=cache(len=0)), mk_.MK_ERR_INVALID, "null cache array")
    refused(f(kv=cache(refs=0)), mk_.MK_ERR_INVALID, "null cache array")
    refused(f(ws=None), mk_.MK_ERR_INVALID, "workspace")
    refused(f(ws=X + 8), mk_.MK_ERR_INVALID, "workspace")
    refused(f(wsb=3), mk_.MK_ERR_INVALID, "workspace")
    refused(f(), mk_.MK_ERR_INVALID, "null context")
    L = mk_.load()
    need = {"fork": L.mk_kv4_fork_workspace(3, 8), "resize": L.mk_kv4_resize_workspace(3, 40),
            "compact": L.mk_kv4_compact_workspace(40)}[f.__name__]
    refused(f(wsb=need - 1), mk_.MK_ERR_INVALID, "workspace")
    refused(f(wsb=need), mk_.MK_ERR_INVALID, "null context")


@pytest.mark.parametrize("over,text", [
    (dict(H=0), "bad sizes"), (dict(pos=-1), "bad sizes"), (dict(layout=2), "layout"), (dict(dim=3), "rope_dim"),
    (dict(dim=130), "rope_dim"), (dict(dim=-2), "rope_dim"), (dict(q=None), "null array"), (dict(k=None), "null array"),
    (dict(v=None), "null array"), (dict(out=None), "null array"), (dict(rpos=None), "null array"), (dict(seq=None), "null array"),
    (dict(row=None), "null array"), (dict(cos=None), "null array"), (dict(sin=None), "null array"), (dict(qn=None), "one norm"),
    (dict(kn=None), "one norm"), (dict(stride=511), "stride"), (dict(os=511), "stride"), (dict(out=X), "other strides"),
    (dict(n=1 << 30), "too many rows"), (dict(), "null context"), (dict(out=X, os=1024), "null context"),
    (dict(dim=0, cos=None, sin=None), "null context"), (dict(qn=None, kn=None), "null context"),
])
def test_rope(over, text):
    refused(rope(**over), mk_.MK_ERR_INVALID, text)


@pytest.mark.parametrize("over,text", [
    (dict(seq=None), "null array"), (dict(row=None), "null array"), (dict(k=X + 8), "aligned"), (dict(v=X + 2), "aligned"),
    (dict(n=1 << 30), "too many rows"), (dict(k=None), "null context"), (dict(v=None), "null context"),
])
def test_rows(over, text):
    refused(rows(**over), mk_.MK_ERR_INVALID, text)


@pytest.mark.parametrize("over,text", [
    (dict(H=0), "bad sizes"), (dict(most=-1), "bad sizes"), (dict(run=-1), "bad sizes"), (dict(H=3), "head layout"),
    (dict(q=None), "null array"), (dict(out=None), "null array"), (dict(seq=None), "null array"), (dict(keys=None), "null array"),
    (dict(qs=511), "stride"), (dict(os=100), "stride"), (dict(n=1 << 23), "too many rows"), (dict(most=257), "past the sequences"),
    (dict(), "null context"), (dict(most=0), "null context"),
])
def test_attention(over, text):
    refused(attention(**over), mk_.MK_ERR_INVALID, text)


def test_attention_heads_and_workspace():
    refused(attention(kv=cache(n_head_kv=1), H=33, qs=33 * 128, os=33 * 128), mk_.MK_ERR_UNSUPPORTED, "head layout")
    L = mk_.load()
    for H, KV, D in ((32, 8, 128), (40, 8, 128), (4, 4, 64), (32, 1, 128)):
        kv = cache(n_head_kv=KV, head_dim=D, max_pages=1 << 14, n_seq=500)
        for run in (1, 5, 100):
            had = 0
            for n in list(range(1, 40)) + [64, 100, 500, 2048]:
                most_need = 0
                for most in (1, 64, 500, 513, 2000, 5000, 40000, 400000):
                    need = L.mk_attention_kv4_workspace(n, H, KV, D, most, run)
                    assert need >= most_need, (n, most)
                    most_need = need
                    a = dict(n=n, H=H, qs=H * D, os=H * D, kv=kv, most=most, run=run)
                    refused(attention(wsb=need, **a), mk_.MK_ERR_INVALID, "null context")
                assert most_need >= had
                had = most_need
    assert L.mk_attention_kv4_workspace(0, 4, 2, 128, 100, 1) == 0
    assert L.mk_attention_kv4_workspace(5, 3, 2, 128, 100, 1) == 0


@pytest.mark.parametrize("f,over,text", [
    (fork, dict(src=None), "null array"), (fork, dict(n=(1 << 20) + 1), "too many entries"), (fork, dict(n=-1), "bad sizes"),
    (resize, dict(len=None), "null array"), (resize, dict(st=None), "null array"), (resize, dict(n=4097), "4096"),
    (resize, dict(n=-1), "bad sizes"), (resize, dict(n=4096), "null context"), (compact, dict(live=None), "null array"),
])
def test_pages(f, over, text):
    refused(f(**over), mk_.MK_ERR_INVALID, text)


@pytest.mark.parametrize("over,text", [
    (dict(groups=-1), "bad sizes"), (dict(V=0), "bad sizes"), (dict(beams=0), "beams"), (dict(beams=65), "beams"), (dict(k=0), "k outside"),
    (dict(k=129), "k outside"), (dict(l=None), "null array"), (dict(s=None), "null array"), (dict(os=None), "null array"),
    (dict(oq=None), "null array"), (dict(ot=None), "null array"), (dict(stride=999), "stride"), (dict(eos=-1), "eos"),
    (dict(eos=1000), "eos"), (dict(V=(1 << 21) + 1, stride=1 << 22), "vocabulary"), (dict(groups=1 << 19), "too many rows"),
    (dict(groups=1 << 17, V=200000, stride=200000), "too many rows"), (dict(ws=None), "workspace"), (dict(wsb=8), "workspace"),
    (dict(ws=X + 4), "workspace"), (dict(), "null context"), (dict(done=None, eos=-7), "null context"),
    (dict(V=1 << 21, stride=1 << 21), "null context"),
])
def test_beam(over, text):
    refused(beam(**over), mk_.MK_ERR_INVALID, text)


def test_empty_calls_and_sizes():
    L = mk_.load()
    assert tables(n=0, cos=None) == mk_.MK_OK and fork(n=0, kv=None) == mk_.MK_OK and resize(n=0, kv=None) == mk_.MK_OK
    assert beam(groups=0, l=None) == mk_.MK_OK
    assert L.mk_kv4_fork_workspace(0, 8) == 0 and L.mk_kv4_resize_workspace(3, 0) == 0 and L.mk_kv4_compact_workspace(0) == 0
    assert L.mk_beam_workspace(1, 65, 1000, 4) == 0 and L.mk_beam_workspace(1, 4, 1000, 129) == 0
    need = L.mk_beam_workspace(2, 4, 1000, 8)
    refused(beam(wsb=need - 1), mk_.MK_ERR_INVALID, "workspace")
    refused(beam(wsb=need), mk_.MK_ERR_INVALID, "null context")
    had = 0
    for g in range(1, 400):  # never less for more groups
        now = L.mk_beam_workspace(g, 4, 151936, 8)
        assert now >= had
        had = now
    assert ctypes.sizeof(mk_.MkKv4Cache) == 88 and ctypes.sizeof(mk_.MkRope) == 56


def test_plain_forms_agree():
    """The model of the cases: numbers in 4 bits stand for values within half a step, and copies leave the source as it is."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((50, 128)).astype(np.float32)
    n, s = cases.in4(x)
    steps = x.reshape(50, 4, 32) / s.astype(np.float64)[..., None]
    far = np.abs(np.clip(steps, -8, 7) - (n.reshape(50, 4, 32).astype(float) - 8))
    assert (far <= 0.5 + 2.0 ** -20).all()
    assert np.array_equal(cases.unpacked(cases.packed(n)), n)
    a = {"table": np.array([[0, 1], [0, 1], [2, -1]], np.int32), "len": np.array([20, 20, 3], np.int32),
         "refs": np.array([2, 2, 1, 0, 0], np.int32)}
    status, copies = cases.resize_model(a, 16, None, [21, 22, 3])
    assert status == [0, 0, 0] and copies == [(1, 3, 4)]
    assert a["table"].tolist() == [[0, 3], [0, 1], [2, -1]] and a["refs"].tolist() == [2, 1, 1, 1, 0]
    cases.fork_model(a, 16, None, [1, 0, -1])
    assert a["table"].tolist() == [[0, 1], [0, 3], [-1, -1]] and a["refs"].tolist() == [2, 1, 0, 1, 0]
    assert cases.compact_model(a) == (3, [(3, 2, None)]) and a["table"].tolist() == [[0, 1], [0, 2], [-1, -1]]


def test_keys_that_are_counted_in_32_bits():
    big = cache(max_pages=1 << 25)
    refused(attention(kv=big, most=(1 << 26) + 1), mk_.MK_ERR_INVALID, "max_keys past 2^26")
    refused(attention(kv=big, most=1 << 26), mk_.MK_ERR_INVALID, "null context")
    refused(attention(kv=cache(n_page=(1 << 27) - 1)), mk_.MK_ERR_INVALID, "null context")
