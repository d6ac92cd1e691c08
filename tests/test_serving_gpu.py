"""GPU: rotary positions, attention over a cache and token sampling through ``CudaBridge``, against ``serving_oracle``."""
import contextlib

import numpy as np
import pytest
import torch

from browsergrad_b200 import HeadView, RotarySpec
from browsergrad_b200.errors import KernelError
from tests import serving_oracle as oracle
from tests.serving_oracle import TORCH

pytestmark = pytest.mark.gpu
DTYPES = ("float32", "float16", "bfloat16")


class Buffers:
    """Uploads and fetches; releases everything at the end."""

    def __init__(self, bridge):
        self.bridge, self.handles = bridge, []

    def put(self, array, dtype):
        if dtype in TORCH:
            t = torch.as_tensor(np.asarray(array)).to(TORCH[dtype]).contiguous()
            raw = t.view(torch.int16 if t.element_size() == 2 else torch.int32).numpy()
        else:
            raw = np.ascontiguousarray(np.asarray(array), dtype=dtype)
        h = self.bridge.upload(raw.tobytes(), np.shape(array), dtype)
        self.handles.append(h)
        return h

    def get(self, handle, shape, dtype):
        raw = self.bridge.materialize(handle, shape, dtype)
        if dtype in TORCH:
            t = torch.frombuffer(bytearray(raw), dtype=TORCH[dtype]) if raw else torch.empty(0, dtype=TORCH[dtype])
            return t.double().numpy().reshape(shape)
        return np.frombuffer(raw, dtype=dtype).reshape(shape)

    def own(self, handle):
        self.handles.append(handle)
        return handle


@pytest.fixture
def buffers(bridge):
    before = bridge.aliveHandleCount()
    b = Buffers(bridge)
    yield b
    with contextlib.suppress(KernelError):
        bridge.synchronize()
    for h in b.handles:
        bridge.release(h)
    assert bridge.aliveHandleCount() == before


def rounded(a, dtype):
    """What the type holds of ``a``, as float64."""
    return torch.as_tensor(np.asarray(a)).to(TORCH[dtype]).double().numpy()


def normal(seed, *shape):
    return np.random.default_rng(seed).standard_normal(shape, dtype=np.float32)


def within(got, want, err, what=""):
    assert got.shape == want.shape
    assert np.isfinite(got).all(), f"{what}: not finite"
    over = np.abs(got - want) - err
    at = np.unravel_index(np.argmax(over), over.shape) if over.size else None
    assert over.size == 0 or over[at] <= 0, f"{what}: {got[at]} against {want[at]} at {at}, bound {err[at]:.3e}"


# -- refusals: on the host, before anything is launched ------------------------------------------------------------------


def test_rotary_refusals(bridge, buffers):
    x = buffers.put(normal(0, 2, 3, 5, 16), "float32")
    half = buffers.put(normal(0, 2, 3, 5, 16), "float16")
    ok = RotarySpec(16)

    def refused(status=1, spec=ok, x=x, b=2, h=3, s=5, d=16, dtype="float32", **kw):
        with pytest.raises(KernelError) as e:
            bridge.rotary(x, spec, b, h, s, d, dtype, **kw)
        assert e.value.status == status, e.value

    refused(spec=RotarySpec(15))
    refused(spec=RotarySpec(18))
    refused(spec=RotarySpec(0))
    refused(spec=RotarySpec(16, base=0.0))
    refused(spec=RotarySpec(16, base=float("nan")))
    refused(spec=RotarySpec(16, scaling="linear", factor=0.0))
    refused(spec=RotarySpec(16, scaling="ramp", factor=2.0, original_length=0.0))
    refused(spec=RotarySpec(16, scaling="ramp", factor=2.0, original_length=8.0, low=4.0, high=4.0))
    refused(spec=RotarySpec(16, magnitude=float("inf")))
    with pytest.raises(KernelError):
        RotarySpec(16, scaling="cubic")
    refused(b=3)
    refused(s=-1)
    refused(b=1 << 40)
    refused(x=half)
    refused(x=10 ** 9, status=5)
    refused(dtype="int32", status=2)
    refused(start=1 << 50)
    refused(positions=x)
    refused(positions=buffers.put(np.zeros(9), "int32"))
    refused(x=HeadView(x, (240, 16, 80), offset=1))
    refused(x=HeadView(x, (240, -16, 80)))
    refused(out=HeadView(x, (240, 80, 16)))                               # x's buffer in another order
    big = buffers.put(np.zeros(1000, np.float32), "float32")
    refused(out=HeadView(big, (240, 8, 80)))                              # rows of the result overlap
    refused(out=HeadView(big, (0, 16, 80)))
    refused(out=big)
    assert bridge.rotary(x, ok, 2, 3, 5, 16, "float32", out=HeadView.heads_first(big, 5, 3, 16)) == big


def test_append_refusals(bridge, buffers):
    q = buffers.put(normal(1, 2, 4, 3, 16), "float32")
    k, v = (buffers.put(normal(s, 2, 2, 3, 16), "float32") for s in (2, 3))
    kc, vc = (buffers.put(np.zeros((2, 2, 8, 16), np.float32), "float32") for _ in range(2))
    ids = buffers.put(np.zeros(2), "int32")

    def refused(q=q, k=k, v=v, kc=kc, vc=vc, s=3, capacity=8, **kw):
        with pytest.raises(KernelError) as e:
            bridge.rotary_append(q, k, v, kc, vc, RotarySpec(16), 2, 4, 2, s, capacity, 16, "float32", **kw)
        assert e.value.status == 1, e.value

    refused(start=6)
    refused(start=-1)
    refused(kc=vc)
    refused(kc=k)
    refused(vc=q)
    refused(out=HeadView.heads_first(q, 3, 4, 16))
    refused(out=HeadView.heads_first(kc, 3, 4, 16))
    refused(capacity=9)
    refused(starts=kc)
    refused(counts=buffers.put(np.zeros(3), "int32"))
    refused(starts=ids, s=4)


@pytest.mark.parametrize("start", [2 ** 63 - 1, 2 ** 63 - 2, 2 ** 62, 2 ** 41])
@pytest.mark.parametrize("counted", [False, True])
def test_append_refuses_a_start_no_cache_has(bridge, buffers, start, counted):
    x = buffers.put(normal(1, 1, 1, 3, 16), "float32")
    caches = [buffers.put(np.zeros((1, 1, 8, 16), np.float32), "float32") for _ in range(2)]
    counts = buffers.put(np.zeros(1), "int32") if counted else None
    with pytest.raises(KernelError) as e:
        buffers.own(bridge.rotary_append(x, x, x, *caches, RotarySpec(16), 1, 1, 1, 3, 8, 16, "float32", start=start, counts=counts))
    assert e.value.status == 1, e.value


def test_attention_refusals(bridge, buffers):
    q = buffers.put(normal(1, 2, 4, 3, 16), "float32")
    k, v = (buffers.put(normal(s, 2, 2, 8, 16), "float32") for s in (2, 3))
    f4, i2, i16 = buffers.put(np.zeros(4), "float32"), buffers.put(np.zeros(2), "int32"), buffers.put(np.zeros(16), "int32")

    def refused(q=q, hq=4, hkv=2, sq=3, sk=8, d=16, status=1, **kw):
        with pytest.raises(KernelError) as e:
            bridge.decoder_attention(q, k, v, 2, hq, hkv, sq, sk, d, "float32", **kw)
        assert e.value.status == status, e.value

    refused(hkv=3)
    refused(hkv=0)
    refused(sk=9)
    refused(softcap=-1.0)
    refused(softcap=float("inf"))
    refused(softcap=1e-20)
    refused(softcap=float("nan"))
    refused(scale=float("nan"))
    refused(scale=1e30)
    refused(prefixes=i2, causal=False)
    refused(slopes=i16)
    refused(documents=i2)
    refused(lengths=f4)
    refused(starts=i16)
    refused(out=HeadView.heads_first(q, 3, 4, 16))
    refused(out=HeadView.heads_first(k, 3, 4, 16))
    refused(d=300, status=2, q=buffers.put(normal(1, 1), "float32"))
    assert bridge.aliveHandleCount() >= 6


def test_sampling_refusals(bridge, buffers):
    x, u = buffers.put(normal(1, 3, 10), "float32"), buffers.put(np.zeros(3), "float32")
    i3, i64 = buffers.put(np.zeros(3), "int32"), buffers.put(np.zeros(3), "int64")

    def refused(x=x, u=u, n=3, vocab=10, status=1, dtype="float32", **kw):
        with pytest.raises(KernelError) as e:
            bridge.sample_tokens(x, u, n, vocab, dtype, **kw)
        assert e.value.status == status, e.value

    refused(temperature=-1.0)
    refused(temperature=float("nan"))
    refused(top_k=-1)
    refused(top_p=float("nan"))
    refused(min_p=-0.1)
    refused(min_p=1.5)
    refused(vocab=11)
    refused(vocab=0)
    refused(u=i3)
    refused(top_ks=u)
    refused(temperatures=i3)
    refused(probabilities=u)
    refused(probabilities=i3)
    refused(out=i3)
    refused(dtype="float64", status=2)
    refused(x=77777777, status=5)
    assert bridge.sample_tokens(x, u, 3, 10, "float32", out=i64) == i64


# -- rotary -----------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,rot,interleaved,kw", [
    (64, 64, False, {}), (128, 128, True, {}), (128, 64, False, dict(scaling="linear", factor=4.0)),
    (80, 40, False, dict(scaling="ramp", factor=8.0, original=512.0, base=500000.0)), (80, 40, True, {}),
    (18, 6, False, {}), (7, 2, True, {}), (256, 256, False, {}), (33, 32, False, dict(magnitude=1.25)), (2, 2, True, {})])
@pytest.mark.parametrize("b,h,s", [(1, 1, 1), (2, 3, 37), (3, 5, 16)])
def test_rotary_matches_the_definition(bridge, buffers, dtype, d, rot, interleaved, kw, b, h, s):
    x = normal(b * 100 + s + d, b, s, h, d)
    pos = np.random.default_rng(d).integers(-5, 200000, (b, s)).astype(np.int32)
    magnitude = kw.get("magnitude", 1.0)
    fkw = {k: v for k, v in kw.items() if k != "magnitude"}
    spec = RotarySpec(rot, base=fkw.get("base", 10000.0), interleaved=interleaved, scaling=fkw.get("scaling", "none"),
                      factor=fkw.get("factor", 1.0), original_length=fkw.get("original", 0.0), magnitude=magnitude)
    hx, hp = buffers.put(x, dtype), buffers.put(pos, "int32")
    xr = rounded(x, dtype)
    for inverse in (False, True):
        want, err = oracle.rotary(xr, pos, oracle.frequencies(rot, **fkw), interleaved, magnitude, inverse)
        out = buffers.own(bridge.rotary(HeadView.rows_first(hx, s, h, d), spec, b, h, s, d, dtype, positions=hp, inverse=inverse))
        got = buffers.get(out, (b, h, s, d), dtype).transpose(0, 2, 1, 3)
        within(got, want, err + oracle.HALF[dtype] * np.abs(want) + (2.0 ** -25 if dtype == "float16" else 0.0), "rotary")
        assert (got[..., rot:] == xr[..., rot:]).all()


@pytest.mark.parametrize("start", [0, -3, 2 ** 31 - 20, 10 ** 12])
def test_rotary_far_positions_keep_their_fraction(bridge, buffers, start):
    b, h, s, d = 1, 2, 9, 64
    x = normal(5, b, h, s, d)
    hx = buffers.put(x, "float32")
    out = buffers.own(bridge.rotary(hx, RotarySpec(d), b, h, s, d, "float32", start=start))
    pos = np.arange(s)[None] + start
    want, err = oracle.rotary(x.astype(np.float64).transpose(0, 2, 1, 3), pos, oracle.frequencies(d))
    within(buffers.get(out, (b, h, s, d), "float32").transpose(0, 2, 1, 3), want, err + 2.0 ** -24 * np.abs(want))


@pytest.mark.parametrize("dtype", DTYPES)
def test_rotary_in_place_on_part_of_a_packed_row_at_an_odd_offset(bridge, buffers, dtype):
    b, s, d = 2, 11, 34
    packed = normal(6, b, s, 3 * d + 1)                   # one value ahead of three heads: nothing is aligned
    h = buffers.put(packed, dtype)
    view = HeadView(h, (s * (3 * d + 1), 3 * d + 1, d), offset=1 + d)          # heads 1 and 2
    assert bridge.rotary(view, RotarySpec(32), b, 2, s, d, dtype, start=4, out=view) == h
    got, src = buffers.get(h, packed.shape, dtype), rounded(packed, dtype)
    x = src[..., 1 + d:].reshape(b, s, 2, d)
    want, err = oracle.rotary(x, np.tile(np.arange(s) + 4, (b, 1)), oracle.frequencies(32))
    within(got[..., 1 + d:].reshape(b, s, 2, d), want, err + oracle.HALF[dtype] * np.abs(want) + 2.0 ** -25)
    assert (got[..., :1 + d] == src[..., :1 + d]).all()


def test_rotary_of_nothing(bridge, buffers):
    x = buffers.put(np.zeros((0, 2, 3, 16), np.float32), "float32")
    out = buffers.own(bridge.rotary(x, RotarySpec(16), 0, 2, 3, 16, "float32"))
    assert buffers.get(out, (0, 2, 3, 16), "float32").size == 0
    out = buffers.own(bridge.rotary(x, RotarySpec(16), 5, 2, 0, 16, "float32"))
    assert buffers.get(out, (5, 2, 0, 16), "float32").size == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,hq,hkv,s,cap,d,rot,interleaved,cache_rows_first", [
    (1, 1, 1, 1, 1, 64, 64, False, False), (3, 4, 2, 7, 20, 64, 32, True, False), (2, 8, 1, 33, 40, 80, 40, False, True),
    (4, 6, 6, 1, 9, 128, 128, False, False), (2, 3, 3, 5, 5, 10, 6, True, True)])
def test_append_writes_new_rows_and_nothing_else(bridge, buffers, dtype, b, hq, hkv, s, cap, d, rot, interleaved, cache_rows_first):
    rng = np.random.default_rng(s * cap)
    qkv = normal(s + cap, b, s, hq + 2 * hkv, d)
    old = [normal(9 + i, b, cap, hkv, d) if cache_rows_first else normal(9 + i, b, hkv, cap, d) for i in range(2)]
    starts = rng.integers(0, cap - s + 1, b).astype(np.int32)
    counts = rng.integers(0, s + 1, b).astype(np.int32)
    h, hs, hc = buffers.put(qkv, dtype), buffers.put(starts, "int32"), buffers.put(counts, "int32")
    caches = [buffers.put(o, dtype) for o in old]
    make = HeadView.rows_first if cache_rows_first else HeadView.heads_first
    n = hq + 2 * hkv
    q, k, v = (HeadView.rows_first(h, s, n, d, first=f) for f in (0, hq, hq + hkv))
    out = buffers.own(bridge.rotary_append(q, k, v, make(caches[0], cap, hkv, d), make(caches[1], cap, hkv, d),
                                           RotarySpec(rot, interleaved=interleaved), b, hq, hkv, s, cap, d, dtype, starts=hs, counts=hc))
    x = rounded(qkv, dtype)
    turned, err = oracle.rotary(x[:, :, :hq + hkv], starts[:, None] + np.arange(s), oracle.frequencies(rot), interleaved)
    err = err + oracle.HALF[dtype] * np.abs(turned) + (2.0 ** -25 if dtype == "float16" else 0.0)
    within(buffers.get(out, (b, hq, s, d), dtype).transpose(0, 2, 1, 3), turned[:, :, :hq], err[:, :, :hq], "q")
    for which in range(2):
        got, before = buffers.get(caches[which], old[which].shape, dtype), rounded(old[which], dtype)
        if not cache_rows_first:
            got, before = got.transpose(0, 2, 1, 3), before.transpose(0, 2, 1, 3)
        for i in range(b):
            a, c = starts[i], counts[i]
            if which == 0:
                within(got[i, a:a + c], turned[i, :c, hq:], err[i, :c, hq:], "k")
            else:
                assert (got[i, a:a + c] == x[i, :c, hq + hkv:]).all()
            assert (got[i, :a] == before[i, :a]).all() and (got[i, a + c:] == before[i, a + c:]).all()
    bridge.synchronize()


@pytest.mark.parametrize("starts,counts", [([6, 0], None), ([-1, 0], None), ([0, 0], [4, 1]), ([0, 0], [-1, 3])])
def test_append_outside_the_cache_is_reported_and_touches_nothing_else(bridge, buffers, starts, counts):
    b, h, s, cap, d = 2, 2, 3, 8, 16
    x = [buffers.put(normal(i, b, h, s, d), "float32") for i in range(3)]
    old = normal(8, b, h, cap, d)
    guard = np.concatenate([normal(7, 64), old.reshape(-1), normal(6, 64)])
    caches = [buffers.put(guard, "float32") for _ in range(2)]
    views = [HeadView(c, (h * cap * d, d, cap * d), offset=64) for c in caches]
    hs = buffers.put(np.asarray(starts), "int32")
    hc = buffers.put(np.asarray(counts), "int32") if counts else None
    out = buffers.own(bridge.rotary_append(*x, *views, RotarySpec(d), b, h, h, s, cap, d, "float32", starts=hs, counts=hc))
    with pytest.raises(KernelError) as e:
        bridge.materialize(out, (b, h, s, d), "float32")
    assert e.value.status == 7
    for c in caches:
        got = buffers.get(c, guard.shape, "float32")
        assert (got[:64] == guard[:64]).all() and (got[-64:] == guard[-64:]).all()


def test_an_append_ends_what_was_kept_about_the_buffers(bridge, buffers):
    """The bridge keeps values derived from a buffer while its handle lives (operand planes of a product); a cache that is
    written in place must not be multiplied by its old planes."""
    m, kk, n = 256, 256, 256
    a, w = normal(1, m, kk), normal(2, kk, n)
    ha, hw = buffers.put(a, "float32"), buffers.put(w, "float32")
    buffers.own(bridge.matmul(ha, hw, m, kk, n, "float32"))
    x = normal(3, 1, 1, kk, n)
    hx, hv = buffers.put(x, "float32"), buffers.put(np.zeros_like(x), "float32")
    buffers.own(bridge.rotary_append(hx, hx, hx, hw, hv, RotarySpec(2), 1, 1, 1, kk, kk, n, "float32"))
    out = buffers.own(bridge.matmul(ha, hw, m, kk, n, "float32"))
    now = buffers.get(hw, (kk, n), "float32")
    want = a.astype(np.float64) @ now
    assert np.abs(buffers.get(out, (m, n), "float32") - want).max() <= 1e-5 * np.abs(want).max()


# -- attention --------------------------------------------------------------------------------------------------------


def run_attention(bridge, buffers, dtype, b, hq, hkv, sq, sk, d, layout="heads", scale=None, seed=0, garbage=True, spread=1.0, **rules):
    """Through the bridge and in 64 bits, with NaN behind every length; returns (got, want, bound)."""
    q, k, v = normal(seed + 1, b, hq, sq, d) * spread, normal(seed + 2, b, hkv, sk, d), normal(seed + 3, b, hkv, sk, d)
    kd, vd = k.copy(), v.copy()
    if garbage and rules.get("lengths") is not None:
        for i, n in enumerate(rules["lengths"]):
            kd[i, :, n:] = np.nan
            vd[i, :, n:] = np.inf

    def place(x):
        heads, rows = x.shape[1], x.shape[2]
        if layout == "heads":
            return HeadView.heads_first(buffers.put(x, dtype), rows, heads, d)
        x = np.ascontiguousarray(x.transpose(0, 2, 1, 3))
        if layout == "rows":
            return HeadView.rows_first(buffers.put(x, dtype), rows, heads, d)
        wide = np.full((b, rows, heads * d + 3), np.nan, np.float32)           # "odd": rows that are never aligned
        wide[:, :, 1:1 + heads * d] = x.reshape(b, rows, heads * d)
        return HeadView(buffers.put(wide, dtype), (rows * (heads * d + 3), heads * d + 3, d), offset=1)

    kw = dict(rules)
    for name, kind in (("slopes", "float32"), ("documents", "int32"), ("prefixes", "int32"), ("lengths", "int32"), ("starts", "int32")):
        if kw.get(name) is not None:
            kw[name] = buffers.put(np.asarray(kw[name]), kind)
    scale = 1 / np.sqrt(d) if scale is None else scale
    out = buffers.own(bridge.decoder_attention(place(q), place(kd), place(vd), b, hq, hkv, sq, sk, d, dtype, scale=scale, **kw))
    got = buffers.get(out, (b, hq, sq, d), dtype)
    want, err = oracle.attention(rounded(q, dtype), rounded(k, dtype), rounded(v, dtype), dtype, scale, **rules)
    return got, want, err


def check_attention(*args, **kw):
    got, want, err = run_attention(*args, **kw)
    within(got, want, err, "attention")


ALIBI = [2.0 ** (-i) for i in range(1, 9)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [16, 40, 64, 72, 80, 96, 128, 200, 256])
@pytest.mark.parametrize("hq,hkv,sq,sk", [(2, 2, 1, 37), (8, 2, 1, 600), (4, 1, 5, 130), (8, 1, 7, 129)])
def test_attention_of_few_rows(bridge, buffers, dtype, d, hq, hkv, sq, sk):
    check_attention(bridge, buffers, dtype, 2, hq, hkv, sq, sk, d, lengths=[sk, max(sq, sk - 19)])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["rows", "odd"])
@pytest.mark.parametrize("d", [64, 96, 128])
def test_attention_layouts(bridge, buffers, dtype, layout, d):
    check_attention(bridge, buffers, dtype, 2, 4, 2, 3, 200, d, layout=layout, lengths=[200, 77])
    check_attention(bridge, buffers, dtype, 2, 4, 2, 150, 150, d, layout=layout, starts=[0, 0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv,s", [(2, 2, 1), (2, 1, 2), (4, 2, 127), (2, 2, 128), (4, 2, 129), (2, 2, 257), (4, 1, 391)])
@pytest.mark.parametrize("rule", ["causal", "both", "capped", "biased", "capped and biased, both", "prefix", "ragged", "documents"])
def test_attention_of_prompts(bridge, buffers, dtype, d, hq, hkv, s, rule):
    b, rng = 2, np.random.default_rng(s)
    kw = dict(starts=[0] * b)
    if "both" in rule:
        kw["causal"] = False
    if "capped" in rule:
        kw["softcap"] = 5.0
    if "biased" in rule:
        kw["slopes"] = ALIBI[:hq]
    if rule == "prefix":
        kw["prefixes"] = [s // 3, s + 10]
    if rule == "ragged":
        kw["lengths"] = [s, s // 2]
    if rule == "documents":
        ids = np.sort(rng.integers(-1, 4, (b, s)), axis=1)
        ids[1] = rng.permutation(ids[1])                 # not even contiguous
        kw["documents"] = ids.astype(np.int32)
    check_attention(bridge, buffers, dtype, b, hq, hkv, s, s, d, spread=3.0, **kw)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("rule", ["plain", "capped", "biased", "prefix, ragged", "both, negative scale"])
def test_attention_of_prompts_beyond_one_tile_a_cta(bridge, buffers, dtype, rule):
    """More than 1024 keys of heads of 64: two query tiles share a CTA and its key tiles."""
    kw = dict(starts=[0], scale=0.2)
    if rule == "capped":
        kw["softcap"] = 8.0
    if rule == "biased":
        kw["slopes"] = [0.03, 0.5]
    if "prefix" in rule:
        kw.update(prefixes=[300], lengths=[1101])
    if "both" in rule:
        kw.update(causal=False, scale=-0.1)
    check_attention(bridge, buffers, dtype, 1, 2, 1, 1155, 1155, 64, spread=2.0, **kw)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_attention_of_prompts_that_end_in_a_late_tile(bridge, buffers, dtype, d):
    """NaN and infinities behind lengths that end in the first to the last of many key tiles."""
    lengths = [1, 129, 300, 511, 640, 777, 901, 1023]
    check_attention(bridge, buffers, dtype, 8, 1, 1, 1024, 1024, d, lengths=lengths, starts=[0] * 8)
    check_attention(bridge, buffers, dtype, 8, 1, 1, 200, 1024, d, lengths=lengths, causal=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [1, 3, 8, 24, 104, 112])
@pytest.mark.parametrize("sq,sk", [(1, 70), (3, 9), (100, 100)])
def test_attention_unusual_head_sizes(bridge, buffers, dtype, d, sq, sk):
    check_attention(bridge, buffers, dtype, 2, 3, 3, sq, sk, d, lengths=[sk, sk - 3], starts=[sk - sq, 0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sq", [1, 90])
def test_attention_with_keys_shared_by_the_batch_and_as_their_own_values(bridge, buffers, dtype, sq):
    """A batch stride of zero, and one buffer for keys and values."""
    b, h, sk, d = 3, 2, 90, 64
    q, k = normal(1, b, h, sq, d), normal(2, 1, h, sk, d)
    hk = buffers.put(k, dtype)
    view = HeadView(hk, (0, d, sk * d))
    out = buffers.own(bridge.decoder_attention(buffers.put(q, dtype), view, view, b, h, h, sq, sk, d, dtype))
    kr = np.broadcast_to(rounded(k, dtype), (b, h, sk, d))
    want, err = oracle.attention(rounded(q, dtype), kr, kr, dtype, 1 / 8)
    within(buffers.get(out, (b, h, sq, d), dtype), want, err)


def test_two_bridges_at_once(bridge, buffers):
    """Calls on two bridges of one device overlap on the GPU; each has its own stream and scratch."""
    from browsergrad_b200 import CudaBridge
    other = CudaBridge(0)
    try:
        mine, theirs = buffers, Buffers(other)
        jobs = []
        for who, bufs in ((bridge, mine), (other, theirs)):
            q, k, v = normal(len(jobs), 1, 4, 2, 64), normal(7 + len(jobs), 1, 2, 9000, 64), normal(9 + len(jobs), 1, 2, 9000, 64)
            jobs.append((who, bufs, [bufs.put(x, "bfloat16") for x in (q, k, v)], (q, k, v), []))
        for _ in range(4):
            for who, bufs, h, _, outs in jobs:
                outs.append(bufs.own(who.decoder_attention(*h, 1, 4, 2, 2, 9000, 64, "bfloat16")))
        for _, bufs, _, (q, k, v), outs in jobs:
            want, err = oracle.attention(*(rounded(x, "bfloat16") for x in (q, k, v)), "bfloat16", 1 / 8)
            for o in outs:
                within(bufs.get(o, (1, 4, 2, 64), "bfloat16"), want, err)
        for h in theirs.handles:
            other.release(h)
        assert other.aliveHandleCount() == 0
    finally:
        other.close()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sq", [1, 4, 200])
def test_attention_rows_that_see_nothing_are_zero(bridge, buffers, dtype, sq):
    b, sk, d = 4, 260, 64
    lengths = [0, 1, sk, 100]
    starts = [0, 0, -3, 95]                               # before the sequence, and behind its end
    got, want, err = run_attention(bridge, buffers, dtype, b, 2, 1, sq, sk, d, lengths=lengths, starts=starts)
    within(got, want, err)
    seen, _ = oracle.visible(b, sq, sk, True, lengths, starts)
    empty = ~seen.any(-1)
    assert empty[0].all() and (got.transpose(0, 2, 1, 3)[empty] == 0).all()
    docs = np.full((b, sk), -1, np.int32)
    got, _, _ = run_attention(bridge, buffers, dtype, b, 2, 1, sq, sk, d, documents=docs, starts=[0] * b)
    assert (got == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,group", [(64, 1), (128, 4)])
@pytest.mark.parametrize("sq", [1, 3, 130])
@pytest.mark.parametrize("softcap", [0.0, 20.0])
def test_attention_bias_of_rows_far_from_their_keys(bridge, buffers, dtype, d, group, sq, softcap):
    # Behind all keys |t - j| = t - j, ahead of them j - t: moving such rows further adds one number to all their scores,
    # which the softmax does not see, so their results are those of rows next to the keys, whatever 32 bits make of slope * t.
    sk, lengths, slopes = 300, [300, 211], np.array(ALIBI[:2 * group], np.float32)
    kw = dict(causal=False, lengths=lengths, slopes=slopes, softcap=softcap, seed=31)
    for near, far in (([300, 211], ([300 + 20_000_003, 211 + 900_001], [2 ** 31 - 1 - sq] * 2)), ([1 - sq] * 2, ([-30_000_001 - sq] * 2, [-2 ** 31] * 2))):
        got, want, err = run_attention(bridge, buffers, dtype, 2, 2 * group, 2, sq, sk, d, starts=near, **kw)
        within(got, want, err, "next to the keys")
        for starts in far:
            moved, _, _ = run_attention(bridge, buffers, dtype, 2, 2 * group, 2, sq, sk, d, starts=starts, **kw)
            assert np.array_equal(moved, got), starts


def test_attention_default_starts_are_the_last_rows(bridge, buffers):
    check_attention(bridge, buffers, "float32", 3, 2, 2, 4, 50, 64, lengths=[50, 4, 2])
    check_attention(bridge, buffers, "bfloat16", 2, 2, 2, 140, 300, 64, lengths=[300, 150])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sq", [2, 140])
def test_attention_without_keys_or_rows(bridge, buffers, dtype, sq):
    q, none = buffers.put(normal(1, 2, 2, sq, 64), dtype), buffers.put(np.zeros((2, 2, 0, 64), np.float32), dtype)
    for causal in (True, False):
        out = buffers.own(bridge.decoder_attention(q, none, none, 2, 2, 2, sq, 0, 64, dtype, causal=causal))
        assert (buffers.get(out, (2, 2, sq, 64), dtype) == 0).all()
    k = buffers.put(normal(1, 2, 2, 9, 64), dtype)
    empty = buffers.put(np.zeros((2, 2, 0, 64), np.float32), dtype)
    out = buffers.own(bridge.decoder_attention(empty, k, k, 2, 2, 2, 0, 9, 64, dtype))
    assert buffers.get(out, (2, 2, 0, 64), dtype).size == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_long_cache_split_over_ctas_repeats_bit_for_bit(bridge, buffers, dtype):
    b, hq, hkv, sq, sk, d = 1, 8, 2, 2, 20011, 128
    first, want, err = run_attention(bridge, buffers, dtype, b, hq, hkv, sq, sk, d, slopes=[0.001 * i for i in range(8)], softcap=20.0)
    within(first, want, err)
    assert bridge.last_plan_trace()[-1].split(" x")[1] not in ("", "1")
    for _ in range(3):
        again, _, _ = run_attention(bridge, buffers, dtype, b, hq, hkv, sq, sk, d, slopes=[0.001 * i for i in range(8)], softcap=20.0)
        assert (again == first).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sq", [1, 130])
def test_attention_large_scores(bridge, buffers, dtype, sq):
    """One key far above the rest, at the end and at the start: the running maximum rises late, or never again."""
    b, h, sk, d = 1, 2, 700, 64
    q = np.ones((b, h, sq, d), np.float32)
    v = normal(4, b, h, sk, d)
    for at in (0, 350, sk - 1):
        k = normal(3, b, h, sk, d) * 0.1
        k[:, :, at] = 8.0
        hq_, hk, hv = buffers.put(q, dtype), buffers.put(k, dtype), buffers.put(v, dtype)
        out = buffers.own(bridge.decoder_attention(hq_, hk, hv, b, h, h, sq, sk, d, dtype, causal=False))
        want, err = oracle.attention(rounded(q, dtype), rounded(k, dtype), rounded(v, dtype), dtype, 1 / 8, causal=False)
        within(buffers.get(out, (b, h, sq, d), dtype), want, err)


def test_attention_length_outside_the_cache_is_reported(bridge, buffers):
    q, k = buffers.put(normal(1, 2, 2, 1, 64), "bfloat16"), buffers.put(normal(2, 2, 2, 30, 64), "bfloat16")
    for lengths in ([31, 5], [5, -1]):
        n = buffers.put(np.asarray(lengths), "int32")
        out = buffers.own(bridge.decoder_attention(q, k, k, 2, 2, 2, 1, 30, 64, "bfloat16", lengths=n))
        with pytest.raises(KernelError) as e:
            bridge.materialize(out, (2, 2, 1, 64), "bfloat16")
        assert e.value.status == 7
    out = buffers.own(bridge.decoder_attention(q, k, k, 2, 2, 2, 1, 30, 64, "bfloat16"))
    assert np.isfinite(buffers.get(out, (2, 2, 1, 64), "bfloat16")).all()


@pytest.mark.parametrize("dtype,apart", [("bfloat16", 1 << 25), ("float32", 1 << 24)])
@pytest.mark.parametrize("odd", [0, 1])
def test_caches_beyond_32_bits_of_offsets(bridge, buffers, dtype, apart, odd):
    # 160 rows `apart` values from each other: the last ones start 5.3 * 10^9 (bfloat16) and 2.7 * 10^9 (float32, 10.7 * 10^9
    # bytes) values into the buffer.  Only strides differ from the dense cache, so results are its bit for bit, as long as
    # both take one kernel: an odd offset keeps TMA out, hence the dense cache starts at it too.
    b, hq, hkv, rows, d = 1, 4, 2, 160, 64
    q, k, v = (buffers.put(normal(40 + i, b, h, rows, d), dtype) for i, h in ((1, hq), (2, hkv), (3, hkv)))
    one = buffers.put(normal(44, b, hq, 1, d), dtype)
    got = []
    for stride in (hkv * d, apart):
        caches = []
        for _ in range(2):
            h = buffers.own(bridge.alloc((odd + (rows - 1) * stride + hkv * d,), dtype))
            caches.append(HeadView(h, (0, stride, d), offset=odd))
        buffers.own(bridge.rotary_append(q, k, v, *caches, RotarySpec(d), b, hq, hkv, rows, rows, d, dtype))
        turned = buffers.own(bridge.rotary(caches[0], RotarySpec(d), b, hkv, rows, d, dtype, start=7))
        got.append([buffers.get(turned, (b, hkv, rows, d), dtype)])
        for rows_q, handle in ((rows, q), (1, one)):
            out = buffers.own(bridge.decoder_attention(handle, *caches, b, hq, hkv, rows_q, rows, d, dtype))
            got[-1].append(buffers.get(out, (b, hq, rows_q, d), dtype))
    for near, far in zip(*got):
        assert np.isfinite(near).all() and np.abs(near).max() > 0.1
        assert np.array_equal(near, far)


def test_a_refused_length_is_reported_ahead_of_a_plans_bytes(bridge, buffers):
    """A plan that brings its result to the host after a refused call must not hand out bytes computed from it."""
    q, k = buffers.put(normal(1, 1, 1, 1, 64), "float32"), buffers.put(normal(2, 1, 1, 9, 64), "float32")
    n = buffers.put(np.asarray([10]), "int32")
    out = buffers.own(bridge.decoder_attention(q, k, k, 1, 1, 1, 1, 9, 64, "float32", lengths=n))
    with pytest.raises(KernelError) as e:
        h = buffers.own(bridge.fused_elementwise([out, out], [("ADD", -1, -2)], (1, 1, 1, 64), "float32"))
        bridge.materialize(h, (1, 1, 1, 64), "float32")
    assert e.value.status == 7
    bridge.synchronize()


# -- sampling ---------------------------------------------------------------------------------------------------------


def run_sample(bridge, buffers, x, u, dtype, chances=True, **kw):
    n, vocab = x.shape
    dev = dict(kw)
    for name, kind in (("temperatures", "float32"), ("top_ks", "int32"), ("top_ps", "float32"), ("min_ps", "float32")):
        if kw.get(name) is not None:
            dev[name] = buffers.put(np.asarray(kw[name]), kind)
    prob = buffers.put(np.full(n, np.nan, np.float32), "float32") if chances else None
    out = buffers.own(bridge.sample_tokens(buffers.put(x, dtype), buffers.put(u, "float32"), n, vocab, dtype, probabilities=prob, **dev))
    return buffers.get(out, (n,), "int64"), buffers.get(prob, (n,), "float32") if chances else None


def check_sample(bridge, buffers, x, u, dtype, **kw):
    got, chance = run_sample(bridge, buffers, x, u, dtype, **kw)
    xr = rounded(x, dtype)
    for i in range(len(x)):
        def one(plural, single, default):
            return kw[plural][i] if kw.get(plural) is not None else kw.get(single, default)
        want, p = oracle.sample(xr[i], u[i], np.float32(one("temperatures", "temperature", 1.0)), int(one("top_ks", "top_k", 0)),
                                one("top_ps", "top_p", 1.0), one("min_ps", "min_p", 0.0))
        assert got[i] == want, (i, got[i], want)
        # the float32 rounding, and the whole-number weights' 2^-47 each against a sum of at least one
        assert abs(chance[i] - p) <= p * (2.0 ** -23 + x.shape[1] * 2.0 ** -46)


def logits(seed, n, vocab):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((n, vocab), dtype=np.float32) * 2
    x[rng.random((n, vocab)) > 0.995] += 6
    return x


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [1, 2, 7, 31, 33, 1000, 4097, 32000, 100003, 200003])
@pytest.mark.parametrize("kw", [{}, dict(top_k=1), dict(top_k=40), dict(top_p=0.9), dict(min_p=0.05), dict(top_p=0.0),
                                dict(top_k=300, top_p=0.7, min_p=0.01, temperature=0.7), dict(temperature=0.0),
                                dict(temperature=3.5, top_p=0.999), dict(top_k=10 ** 9)])
def test_sampling_matches_the_definition(bridge, buffers, dtype, vocab, kw):
    n = 5
    u = np.random.default_rng(vocab).random(n, dtype=np.float32)
    u[0], u[1] = 0.0, np.float32(1 - 2.0 ** -24)
    check_sample(bridge, buffers, logits(vocab, n, vocab), u, dtype, **kw)


@pytest.mark.parametrize("top_k", [5, 127, 128, 129, 256, 257, 3000, 39999])
@pytest.mark.parametrize("top_p", [1.0, 0.6])
def test_sampling_of_many_ranks(bridge, buffers, top_k, top_p):
    """From the list of the threads' own maxima to the general threshold, over values with ties at every rank."""
    x = rounded(logits(9, 3, 40000), "float16")
    x[1] = np.round(x[1])
    x[2, 100:] = -np.inf                     # fewer candidates than ranks
    check_sample(bridge, buffers, x, np.array([0.2, 0.7, 0.95], np.float32), "float16", top_k=top_k, top_p=top_p)


def test_sampling_of_a_large_batch(bridge, buffers):
    """Several rounds of clusters on the device, one and several CTAs a row."""
    for n, vocab in ((600, 3000), (170, 33001)):
        check_sample(bridge, buffers, logits(n, n, vocab), np.random.default_rng(n).random(n, dtype=np.float32), "bfloat16", top_p=0.9, top_k=0)


@pytest.mark.parametrize("vocab", [64, 5000, 60001])
def test_sampling_parameters_per_row(bridge, buffers, vocab):
    n, rng = 24, np.random.default_rng(vocab)
    check_sample(bridge, buffers, logits(1, n, vocab), rng.random(n, dtype=np.float32), "bfloat16",
                 temperatures=rng.choice([0.0, 0.3, 1.0, 2.0], n).astype(np.float32), top_ks=rng.choice([0, 1, 5, 100, -2], n),
                 top_ps=rng.choice([0.1, 0.5, 0.95, 1.0, 2.0], n).astype(np.float32), min_ps=rng.choice([0.0, 0.01, 0.5], n).astype(np.float32))


@pytest.mark.parametrize("vocab", [40, 3000, 70000])
@pytest.mark.parametrize("kw", [dict(top_k=7), dict(top_p=0.3), dict(top_k=20, top_p=0.55), dict(), dict(min_p=1.0), dict(top_k=1)])
def test_sampling_takes_equal_logits_in_index_order(bridge, buffers, vocab, kw):
    """Few distinct values, so that every threshold falls among equal ones; rows of one value alone; signed zeros."""
    rng = np.random.default_rng(vocab)
    x = rng.integers(-2, 3, (6, vocab)).astype(np.float32)
    x[1] = 4.0
    x[2] = np.where(rng.random(vocab) < 0.5, -0.0, 0.0)
    x[3] = -3.0e38
    x[4, 1:] = -3.0e38
    u = rng.random(6, dtype=np.float32)
    check_sample(bridge, buffers, x, u, "float32", **kw)


@pytest.mark.parametrize("kw", [{}, dict(top_k=3), dict(top_p=0.8), dict(min_p=0.1), dict(temperature=0.0)])
def test_sampling_rows_with_infinities_and_nan(bridge, buffers, kw):
    vocab = 300
    x = logits(3, 7, vocab)
    x[0] = -np.inf
    x[1] = np.nan
    x[2, ::2] = -np.inf
    x[3, 5], x[3, 17] = np.inf, np.inf
    x[4, :] = -np.inf
    x[4, 123] = -50.0
    x[5, 40:60] = np.nan
    x[6, :] = np.finfo(np.float32).min
    check_sample(bridge, buffers, x, np.random.default_rng(1).random(7, dtype=np.float32), "float32", **kw)


def test_sampling_extreme_temperatures_and_numbers_outside_the_range(bridge, buffers):
    x = logits(5, 6, 1000)
    t = np.array([1e-30, 1e30, np.float32(1e-45), 0.5, 0.5, -1.0], np.float32)
    u = np.array([0.5, 0.25, 0.9, -0.5, 1.0, 0.3], np.float32)
    check_sample(bridge, buffers, x, u, "float32", temperatures=t)


def test_sampling_follows_the_distribution_and_repeats(bridge, buffers):
    """4096 draws of one row with evenly spaced numbers hit each token in proportion, to within one draw: a token whose
    interval has length p holds between floor(4096 p) and ceil(4096 p) + 1 of the points."""
    vocab, n = 50, 4096
    row = np.linspace(-2, 2, vocab, dtype=np.float32)
    x = np.tile(row, (n, 1))
    u = (np.arange(n) / n).astype(np.float32)
    got, _ = run_sample(bridge, buffers, x, u, "float32")
    p = np.exp(row.astype(np.float64))
    p /= p.sum()
    hits = np.bincount(got, minlength=vocab)
    assert (np.abs(hits - n * p) <= 1 + 1e-6).all()
    again, _ = run_sample(bridge, buffers, x, u, "float32", chances=False)
    assert (again == got).all()


def test_sampling_of_no_rows(bridge, buffers):
    got, _ = run_sample(bridge, buffers, np.zeros((0, 9), np.float32), np.zeros(0, np.float32), "float32")
    assert got.shape == (0,)


# -- together ---------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_generation_loop(bridge, buffers, dtype):
    """Prompts of different lengths enter the cache, then tokens are generated one by one: rotary_append,
    decoder_attention over the cache, the product with an output matrix, sample_tokens, and the token's embedding is the
    next input.  Each step's attention is compared with the whole sequence computed at once from the same inputs."""
    b, hq, hkv, d, cap, vocab, steps = 3, 4, 2, 64, 48, 257, 6
    n = hq + 2 * hkv
    rng = np.random.default_rng(11)
    embed = (normal(21, vocab, n * d) * 0.5)
    head = normal(22, hq * d, vocab) * 0.2
    prompt = np.array([7, 1, 12], np.int32)
    spec, f = RotarySpec(d), oracle.frequencies(d)
    ids = rng.integers(0, vocab, (b, int(prompt.max())))
    kc, vc = (buffers.put(np.full((b, hkv, cap, d), np.nan, np.float32), dtype) for _ in range(2))
    hw = buffers.put(head, "float32")
    history = [[] for _ in range(b)]                  # the inputs of every position, as the device saw them
    starts, counts, s = np.zeros(b, np.int32), prompt.copy(), ids.shape[1]
    tokens = ids
    for step in range(steps):
        x = embed[tokens].reshape(b, s, n, d)
        xr = rounded(x, dtype)
        for i in range(b):
            history[i] += list(xr[i, :counts[i]])
        h = buffers.put(x, dtype)
        q, k, v = (HeadView.rows_first(h, s, n, d, first=g) for g in (0, hq, hq + hkv))
        hs, hc, hl = buffers.put(starts, "int32"), buffers.put(counts, "int32"), buffers.put(starts + counts, "int32")
        turned = buffers.own(bridge.rotary_append(q, k, v, kc, vc, spec, b, hq, hkv, s, cap, d, dtype, starts=hs, counts=hc))
        out = buffers.put(np.zeros((b, s, hq, d), np.float32), dtype)
        bridge.decoder_attention(turned, kc, vc, b, hq, hkv, s, cap, d, dtype, softcap=20.0, lengths=hl, starts=hs,
                                 out=HeadView.rows_first(out, s, hq, d))
        got = buffers.get(out, (b, s, hq, d), dtype)
        last = np.stack([got[i, counts[i] - 1].reshape(-1) for i in range(b)])
        for i in range(b):
            seq = np.stack(history[i])[None]
            pos = np.arange(seq.shape[1])[None]
            qk, _ = oracle.rotary(seq[:, :, :hq + hkv], pos, f)
            qk = rounded(qk, dtype).transpose(0, 2, 1, 3)     # the caches hold the operand type
            want, err = oracle.attention(qk[:, :hq, -counts[i]:], qk[:, hq:], seq[:, :, hq + hkv:].transpose(0, 2, 1, 3), dtype, 1 / 8, softcap=20.0)
            # a rotated value next to a rounding border may go to the other side on the device: half a step more, twice (q
            # and k), of the largest product
            slack = 4 * oracle.HALF[dtype] * np.abs(want).max()
            within(got[i, :counts[i]], want[0].transpose(1, 0, 2), err[0].transpose(1, 0, 2) + slack, f"step {step}")
        logit = buffers.own(bridge.matmul(buffers.put(last, "float32"), hw, b, hq * d, vocab, "float32"))
        u = rng.random(b, dtype=np.float32)
        drawn = buffers.own(bridge.sample_tokens(logit, buffers.put(u, "float32"), b, vocab, "float32", temperature=0.8, top_k=40, top_p=0.9))
        z = buffers.get(logit, (b, vocab), "float32")
        tokens = buffers.get(drawn, (b,), "int64")
        assert [oracle.sample(z[i], u[i], np.float32(0.8), 40, 0.9)[0] for i in range(b)] == list(tokens)
        starts, counts, s, tokens = starts + counts, np.ones(b, np.int32), 1, tokens[:, None]


def test_calls_into_a_captured_stream_are_refused(bridge, buffers):
    x, u = buffers.put(normal(1, 2, 2, 3, 64), "float32"), buffers.put(np.zeros(2), "float32")
    lg = buffers.put(normal(2, 2, 9), "float32")
    bridge.synchronize()
    graph = torch.cuda.CUDAGraph()
    stream = torch.cuda.ExternalStream(bridge.stream())
    calls = [lambda: bridge.rotary(x, RotarySpec(64), 2, 2, 3, 64, "float32"),
             lambda: bridge.decoder_attention(x, x, x, 2, 2, 2, 3, 3, 64, "float32"),
             lambda: bridge.sample_tokens(lg, u, 2, 9, "float32")]
    got = []
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="relaxed"):
        for call in calls:
            try:
                call()
                got.append(None)
            except KernelError as e:
                got.append(e.status)
    assert got == [2, 2, 2]
    del graph
    for call in calls:
        buffers.own(call())
    bridge.synchronize()


def test_profiles_and_the_trace_name_the_operators(bridge, buffers):
    x = buffers.put(normal(1, 1, 2, 3, 64), "float32")
    bridge.set_option("profiling", 1)
    try:
        launches = bridge.resourceSnapshot()["kernelLaunches"]
        buffers.own(bridge.rotary(x, RotarySpec(64), 1, 2, 3, 64, "float32"))
        assert bridge.last_plan_trace() == ["rotary[float32]"]
        buffers.own(bridge.decoder_attention(x, x, x, 1, 2, 2, 3, 3, 64, "float32"))
        assert bridge.resourceSnapshot()["kernelLaunches"] == launches + 2
        names = {p["name"] for p in bridge.flushProfiles()}
        assert "rotary[float32]" in names and any(n.startswith("cache_attention[float32]") for n in names)
    finally:
        bridge.set_option("profiling", 0)


def test_failed_allocations_leave_no_handles(bridge, buffers):
    x = buffers.put(normal(1, 1, 2, 300, 64), "bfloat16")
    docs = buffers.put(np.zeros((1, 300)), "int32")
    before = bridge.aliveHandleCount()
    for nth in (1, 2):
        bridge.set_option("fail_allocation_after", nth)
        try:
            with pytest.raises(KernelError) as e:
                bridge.decoder_attention(x, x, x, 1, 2, 2, 300, 300, 64, "bfloat16", documents=docs)
            assert e.value.status == 4
        finally:
            bridge.set_option("fail_allocation_after", 0)
    assert bridge.aliveHandleCount() == before
