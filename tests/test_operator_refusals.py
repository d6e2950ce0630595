"""Arguments that the shared-prefix attention, adapter and verification calls refuse, before anything touches a device
(the context is the last thing they look at, so no GPU is needed), and the sizes that their workspaces report."""
import ctypes

import numpy as np
import pytest

import malkin_amd as mk_

X = 1 << 20  # a 16-byte aligned address that nothing reads


def refused(rc, code, text):
    assert rc == code, rc
    assert text in mk_.load().mk_last_error().decode(), mk_.load().mk_last_error()


def cache(**over):
    f = dict(k=X, v=X, k_scale=X, v_scale=X, n_layer=2, n_seq=3, n_head_kv=2, head_dim=128, n_ctx=64)
    f.update(over)
    return mk_.MkKvCache(*(f[n] for n, _ in mk_.MkKvCache._fields_))


def prefix_call(**over):
    L = mk_.load()
    a = dict(q=X, qs=512, out=X, os=512, n=5, H=4, pre=cache(), pseq=1, P=40, kv=cache(), row0=0, layer=1, seq=X,
             keys=X, most=100, xq=None, ws=X, wsb=1 << 30)
    a.update(over)
    ref = [ctypes.byref(a[x]) if a[x] is not None else None for x in ("pre", "kv")]
    return L.mk_attention_prefix(None, a["q"], a["qs"], a["out"], a["os"], a["n"], a["H"], ref[0], a["pseq"], a["P"],
                                 ref[1], a["row0"], a["layer"], a["seq"], a["keys"], a["most"], a["xq"], a["ws"],
                                 a["wsb"])


@pytest.mark.parametrize("over,text", [
    (dict(n=-1), "bad sizes"), (dict(H=0), "bad sizes"), (dict(P=-1), "bad sizes"), (dict(row0=-1), "bad sizes"),
    (dict(most=-1), "bad sizes"), (dict(kv=None), "bad KV cache"), (dict(layer=2), "bad KV cache"),
    (dict(layer=-1), "bad KV cache"), (dict(H=3), "bad head layout"), (dict(q=None), "null array"),
    (dict(out=None), "null array"), (dict(seq=None), "null array"), (dict(keys=None), "null array"),
    (dict(qs=511), "stride"), (dict(os=100), "stride"), (dict(most=105), "past the sequence's rows"),
    (dict(row0=5), "past the sequence's rows"), (dict(n=1 << 29), "too many rows"),
    (dict(kv=cache(k=X + 8)), "16-byte aligned"), (dict(kv=cache(v=0)), "16-byte aligned"),
    (dict(kv=cache(v_scale=0)), "16-byte aligned"), (dict(pre=None), "bad KV cache"),
    (dict(pre=cache(n_layer=1)), "bad KV cache"), (dict(pre=cache(n_head_kv=1)), "other heads"),
    (dict(pre=cache(head_dim=64)), "other heads"), (dict(pseq=3), "outside its cache"),
    (dict(pseq=-1), "outside its cache"), (dict(pre=cache(n_ctx=39)), "outside its cache"),
    (dict(pre=cache(v=X + 4)), "16-byte aligned"), (dict(), "null context"),
])
def test_prefix_refusals(over, text):
    refused(prefix_call(**over), mk_.MK_ERR_INVALID, text)


def test_prefix_unsupported():
    for kv in (cache(head_dim=96), cache(head_dim=32)):
        refused(prefix_call(kv=kv, pre=kv), mk_.MK_ERR_UNSUPPORTED, "no kernel")
    one = cache(n_head_kv=1)
    refused(prefix_call(kv=one, pre=one, H=33, qs=33 * 128, os=33 * 128), mk_.MK_ERR_UNSUPPORTED, "no kernel")


def test_prefix_workspace():
    L = mk_.load()
    need = L.mk_attention_prefix_workspace(5, 4, 2, 128, 40, 100)
    if need:
        refused(prefix_call(wsb=need - 1), mk_.MK_ERR_INVALID, "workspace")
        refused(prefix_call(ws=X + 4), mk_.MK_ERR_INVALID, "workspace")
        refused(prefix_call(ws=None), mk_.MK_ERR_INVALID, "workspace")
    refused(prefix_call(wsb=need), mk_.MK_ERR_INVALID, "null context")
    assert L.mk_attention_prefix_workspace(0, 4, 2, 128, 40, 100) == 0
    assert L.mk_attention_prefix_workspace(5, 3, 2, 128, 40, 100) == 0
    # No tokens: nothing to do, whatever the rest says.
    assert prefix_call(n=0, kv=None) == mk_.MK_OK


def lora_call(**over):
    a = dict(type=mk_.F16, table=X, na=3, rank=16, ids=X, x=X, xs=256, n=4, rows=512, cols=256, base=X, bs=512, y=X + 64,
             ys=512, ws=X, wsb=1 << 30)
    a.update(over)
    return mk_.load().mk_lora(None, *a.values())


@pytest.mark.parametrize("over,text", [
    (dict(n=-1), "bad sizes"), (dict(na=-1), "bad sizes"), (dict(rows=0), "bad sizes"), (dict(cols=0), "bad sizes"),
    (dict(rank=0), "max_rank"), (dict(rank=513), "max_rank"), (dict(rows=1 << 25, ys=1 << 25, bs=1 << 25), "too large"),
    (dict(x=None), "null array"), (dict(y=None), "null array"), (dict(ids=None), "null array"),
    (dict(table=None), "null array"), (dict(xs=255), "stride"), (dict(ys=511), "stride"), (dict(bs=511), "stride"),
    (dict(base=X, y=X, bs=520), "other strides"), (dict(ws=None), "workspace"), (dict(wsb=8), "workspace"),
    (dict(ws=X + 8), "workspace"), (dict(), "null context"), (dict(base=None), "null context"),
    (dict(table=None, na=0), "null context"),
])
def test_lora_refusals(over, text):
    refused(lora_call(**over), mk_.MK_ERR_INVALID, text)


def test_lora_types():
    for t in (mk_.Q8_0, mk_.Q4_K, 5):
        refused(lora_call(type=t), mk_.MK_ERR_UNSUPPORTED, "F32, F16 or BF16")
    need = mk_.load().mk_lora_workspace(4, 16, 256)
    refused(lora_call(wsb=need - 1), mk_.MK_ERR_INVALID, "workspace")
    refused(lora_call(wsb=need), mk_.MK_ERR_INVALID, "null context")
    assert lora_call(n=0, x=None) == mk_.MK_OK


def verify_call(**over):
    a = dict(p=X, ps=1000, rows=9, q=X, qs=1000, drafts=6, V=1000, lanes=X, nl=3, most=4, d=X, u=X, un=X, acc=X, tok=X,
             pr=None, ws=X, wsb=1 << 30)
    a.update(over)
    return mk_.load().mk_verify(None, *a.values())


@pytest.mark.parametrize("over,text", [
    (dict(rows=-1), "bad sizes"), (dict(drafts=-1), "bad sizes"), (dict(nl=-1), "bad sizes"),
    (dict(most=-1), "max_draft"), (dict(most=257), "max_draft"), (dict(nl=1 << 29, most=2), "too many lanes"),
    (dict(lanes=None), "null array"), (dict(un=None), "null array"), (dict(acc=None), "null array"),
    (dict(tok=None), "null array"), (dict(d=None), "null array"), (dict(u=None), "null array"),
    (dict(p=None), "null array"), (dict(V=0), "bad vocabulary"), (dict(ps=999), "stride"), (dict(qs=999), "stride"),
    (dict(ws=None), "workspace"), (dict(wsb=100), "workspace"), (dict(ws=X + 4), "workspace"),
    (dict(), "null context"), (dict(q=None, qs=0), "null context"), (dict(drafts=0, d=None, u=None), "null context"),
])
def test_verify_refusals(over, text):
    refused(verify_call(**over), mk_.MK_ERR_INVALID, text)


def topk_call(**over):
    a = dict(pv=X, pi=X, pk=40, rows=9, qv=X, qi=X, qk=40, drafts=6, lanes=X, nl=3, most=4, d=X, u=X, un=X, acc=X, tok=X,
             pr=None)
    a.update(over)
    return mk_.load().mk_verify_topk(None, *a.values())


@pytest.mark.parametrize("over,text", [
    (dict(pk=0), "1..1024"), (dict(pk=1025), "1..1024"), (dict(qk=0), "1..1024"), (dict(qk=1025), "1..1024"),
    (dict(qi=None), "without ids"), (dict(qv=None), "without ids"), (dict(pv=None), "null array"),
    (dict(pi=None), "null array"), (dict(tok=None), "null array"), (dict(most=257), "max_draft"),
    (dict(nl=-1), "bad sizes"), (dict(), "null context"), (dict(qv=None, qi=None, qk=0), "null context"),
])
def test_verify_topk_refusals(over, text):
    refused(topk_call(**over), mk_.MK_ERR_INVALID, text)


def test_empty_calls_and_tables():
    L = mk_.load()
    assert verify_call(nl=0, lanes=None, un=None, acc=None, tok=None) == mk_.MK_OK
    assert topk_call(nl=0, lanes=None, un=None, acc=None, tok=None) == mk_.MK_OK
    assert L.mk_verify_workspace(0, 4, 1000) == 0 and L.mk_verify_workspace(3, -1, 1000) == 0
    assert L.mk_verify_workspace(3, 4, 1000) > 0
    assert L.mk_lora_workspace(0, 16, 256) == 0
    # The tables' Python layouts are the header's.
    assert mk_.LORA_ADAPTER.itemsize == 24 and mk_.VERIFY_LANE.itemsize == 24
    assert np.zeros(1, mk_.LORA_ADAPTER).dtype.fields["rank"][1] == 20


@pytest.mark.parametrize("H,KV,D", [(32, 8, 128), (40, 8, 128), (4, 4, 64), (16, 1, 128)])
def test_prefix_workspace_holds_smaller_calls(H, KV, D):
    """A workspace for a number of tokens and a bound on the keys is enough for every smaller one, and no call asks for
    more than its own sizes report."""
    L = mk_.load()
    kv, few = (cache(n_head_kv=KV, head_dim=D, n_ctx=20000, n_seq=m) for m in (300, 1))
    for P in (0, 100, 2048, 9000):
        had = 0
        for n in list(range(1, 70)) + [100, 127, 128, 129, 255, 256, 257, 400, 512, 513, 1024, 1100, 4096]:
            row, most_need = [], 0
            for most in (P // 2, P, P + 1, P + 128, P + 129, P + 1024, P + 6200):
                row.append(L.mk_attention_prefix_workspace(n, H, KV, D, P, most))
                assert row[-1] >= most_need, (P, n, most)
                most_need = row[-1]
                for own in (kv, few):
                    refused(prefix_call(n=n, H=H, qs=H * D, os=H * D, kv=own, pre=kv, P=P, most=most, wsb=row[-1]),
                            mk_.MK_ERR_INVALID, "null context")
            assert row[-1] >= had, (P, n)
            had = row[-1]
            # Not a multiple of what the call uses: at most 64 parts of a row.
            assert row[-1] <= 64 * n * H * (4 * D + 16)


def test_lora_workspace_holds_smaller_calls():
    L = mk_.load()
    for cols in (32, 512, 1000, 4096, 20000):
        had = 0
        for n in range(1, 20000, 7):
            need = L.mk_lora_workspace(n, 16, cols)
            assert need >= had and need <= 16 * n * 16 * 4, (cols, n)
            had = need
            if n % 50 == 1:
                refused(lora_call(n=n, cols=cols, xs=cols, wsb=need), mk_.MK_ERR_INVALID, "null context")
        assert L.mk_lora_workspace(100, 16, cols) <= L.mk_lora_workspace(100, 64, cols) <= \
            L.mk_lora_workspace(100, 64, 2 * cols)


@pytest.mark.parametrize("over", [dict(rows=-1), dict(most=257), dict(nl=1 << 29), dict(lanes=None), dict(d=None)])
def test_refusals_name_their_call(over):
    for call, name in ((verify_call, "mk_verify: "), (topk_call, "mk_verify_topk: ")):
        assert call(**over) == mk_.MK_ERR_INVALID
        assert mk_.load().mk_last_error().decode().startswith(name)


def test_prefix_launch_limits():
    """A launch has fewer than 2^32 threads."""
    one = cache(n_head_kv=1, head_dim=64, n_ctx=200)
    a = dict(H=1, qs=64, os=64, kv=one, pre=None, P=0, most=100, wsb=1 << 50)
    refused(prefix_call(n=1 << 24, **a), mk_.MK_ERR_INVALID, "too many rows")
    refused(prefix_call(n=(1 << 24) - 64, **a), mk_.MK_ERR_INVALID, "null context")
    wide = cache(n_head_kv=8)
    a = dict(H=256, qs=1 << 15, os=1 << 15, kv=wide, pre=wide, P=40, most=40, wsb=1 << 50)
    refused(prefix_call(n=1 << 18, **a), mk_.MK_ERR_INVALID, "too many rows")
    refused(prefix_call(n=(1 << 18) - 1, **a), mk_.MK_ERR_INVALID, "null context")


def test_lora_launch_limits():
    """A launch has fewer than 2^32 threads, and no count wraps on the way there."""
    a = dict(cols=1, xs=1, rank=1, rows=1, ys=1, bs=1, wsb=1 << 60)
    for n in (1 << 29, (1 << 31) - 64, (1 << 31) - 1):
        refused(lora_call(n=n, **a), mk_.MK_ERR_INVALID, "too many tokens")
        assert mk_.load().mk_lora_workspace(n, 1, 1) == 64 * n
    refused(lora_call(n=(1 << 29) - 64, **a), mk_.MK_ERR_INVALID, "null context")
    a.update(rows=1 << 24, ys=1 << 24, bs=1 << 24)
    refused(lora_call(n=1 << 14, **a), mk_.MK_ERR_INVALID, "too many tokens")
    refused(lora_call(n=(1 << 14) - 64, **a), mk_.MK_ERR_INVALID, "null context")


def test_verify_launch_limits():
    """A launch has fewer than 2^32 threads."""
    a = dict(most=0, drafts=0, d=None, u=None, wsb=1 << 60)
    refused(verify_call(nl=1 << 24, **a), mk_.MK_ERR_INVALID, "too many lanes")
    refused(verify_call(nl=(1 << 24) - 1, **a), mk_.MK_ERR_INVALID, "null context")
    # 257 + 256 rows a lane, of 2^27 logits each: 4096 workgroups a row.
    a = dict(most=256, rows=1 << 20, drafts=1 << 20, V=1 << 27, ps=1 << 27, qs=1 << 27, wsb=1 << 60)
    refused(verify_call(nl=8, **a), mk_.MK_ERR_INVALID, "too many lanes")
    refused(verify_call(nl=7, **a), mk_.MK_ERR_INVALID, "null context")
    a = dict(most=0, drafts=0, d=None, u=None)
    refused(topk_call(nl=1 << 23, **a), mk_.MK_ERR_INVALID, "too many lanes")
    refused(topk_call(nl=(1 << 23) - 1, **a), mk_.MK_ERR_INVALID, "null context")


def test_prefix_row_past_32_bits():
    """The kernels' offsets inside a token's row are 32-bit."""
    kv = cache(n_head_kv=1 << 20, n_ctx=41)
    a = dict(n=1, kv=kv, pre=kv, P=40, most=41, qs=1 << 40, os=1 << 40, wsb=1 << 50)
    refused(prefix_call(H=1 << 24, **a), mk_.MK_ERR_INVALID, "bad head layout")
    refused(prefix_call(H=(1 << 24) - (1 << 20), **a), mk_.MK_ERR_INVALID, "null context")
