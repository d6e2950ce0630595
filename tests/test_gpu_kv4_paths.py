"""Attention over the 4-bit cache by each of its kernels, and with scales among fp16's subnormal numbers."""
import numpy as np
import pytest

import malkin_amd as mk_
from kv4_cases import attention64
from kv4_paths import CASES, path_of
from test_gpu_kv4 import Call, build, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in c[:4] + path_of(c)))
def test_attention(mk, case):
    H, KV, d, page, new, rows = case
    rng = np.random.default_rng(sum(new) + max(rows))
    c, q, seq, keys = build(rng, H, KV, d, page, new, rows, 1)
    c.put(mk)
    want = attention64(c, 0, q, H, seq, keys)
    print("kv4 attention, paths", case[:4], path_of(case), flush=True)
    call = Call(mk, c, q, H, 0, seq, keys, max(keys), max(new), 3, True)
    call.run()
    got = call.result()
    check(got, want)
    ref, dense = mk.alloc(call.n * call.HD // 32 * 40), mk.to_device(got)
    mk_.check(mk_.load().mk_quantize_q8(mk.h, dense.ptr, call.n, call.HD, ref.ptr))
    assert np.array_equal(ref.download(np.uint8), call.xq.download(np.uint8))
    call.run()
    assert np.array_equal(got.view(np.uint32), call.result().view(np.uint32))


@pytest.mark.parametrize("H,KV,d,new,rows", [(8, 2, 128, 1, 300), (8, 2, 64, 7, 130), (16, 2, 128, 40, 700), (4, 2, 64, 1, 5000)])
@pytest.mark.parametrize("side", ["k", "v", "kv"])
def test_subnormal_scales(mk, H, KV, d, new, rows, side):
    """Scales of at most 255 steps of 2^-24, as a head whose values are all below 5e-4 has them: what the numbers stand for is
    exact in fp16 (11 bits), but subnormal where it is below 2^-14."""
    rng = np.random.default_rng(rows)
    c, q, seq, keys = build(rng, H, KV, d, 16, [new] * 3, [rows, new + 1, 77], 1)
    for x in side:
        s = rng.integers(-255, 256, c.a[x + "_scale"].shape) * 2.0 ** -24
        c.a[x + "_scale"] = s.astype(np.float16)
        assert (np.abs(c.a[x + "_scale"].astype(np.float64)) <= 255 * 2.0 ** -24).all() and (c.a[x + "_scale"] == s).all()
    q *= 2000  # scores that differ
    c.put(mk)
    want = attention64(c, 0, q, H, seq, keys)
    assert np.abs(want[0]).max() > 0
    call = Call(mk, c, q, H, 0, seq, keys, max(keys), new)
    print("kv4 attention, subnormal scales", H, d, new, rows, side, flush=True)
    call.run()
    check(call.result(), want, norm=False)
