"""GPU: the serving operators at the ends of what they accept, against ``serving_oracle``."""
from concurrent.futures import ThreadPoolExecutor

import numpy as np
import pytest

from browsergrad_b200 import HeadView, RotarySpec
from browsergrad_b200.errors import KernelError
from tests import serving_oracle as oracle
from tests.test_serving_gpu import DTYPES, buffers, normal, rounded, run_sample, within  # noqa: F401  (buffers is a fixture)

pytestmark = pytest.mark.gpu


def attend(bridge, buffers, dtype, q, k, v, **rules):
    """[b, heads, rows, d] arrays through the bridge; index rules are given as arrays."""
    (b, hq, sq, d), (_, hkv, sk, _) = q.shape, k.shape
    dev = {n: buffers.put(np.asarray(x), "int32") if n in ("lengths", "starts", "prefixes", "documents") else x for n, x in rules.items()}
    out = buffers.own(bridge.decoder_attention(*(buffers.put(x, dtype) for x in (q, k, v)), b, hq, hkv, sq, sk, d, dtype, **dev))
    return buffers.get(out, (b, hq, sq, d), dtype)


def expected(dtype, q, k, v, smallest=2.0 ** -25, **rules):
    q, k, v = (rounded(x, dtype) for x in (q, k, v))
    scale = rules.pop("scale", 1 / np.sqrt(q.shape[-1]))
    want, _ = oracle.attention(q, k, v, dtype, scale, **rules)
    return want, oracle.attention_bound(q, k, v, want, dtype, scale, smallest=smallest, **rules)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("sq", [1, 63, 64, 200])
@pytest.mark.parametrize("softcap", [1e3, 1e5, 1e6])
def test_attention_caps_far_above_the_scores(bridge, buffers, dtype, d, sq, softcap):
    """A cap that hardly bends the scores must not cost them their digits."""
    q, k, v = normal(1, 2, 4, sq, d) * 1.5, normal(2, 2, 2, 300, d), normal(3, 2, 2, 300, d)
    rules = dict(lengths=[300, 211], softcap=softcap)
    within(attend(bridge, buffers, dtype, q, k, v, **rules), *expected(dtype, q, k, v, **rules))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("sq", [9, 64, 200])
def test_attention_rows_beyond_the_cap_next_to_rows_far_below_it(bridge, buffers, dtype, sq):
    """Every eighth row's scores pass the cap (their exponents are off by about one in 32 bits: only finite), the others are a
    millionth of it and keep their digits."""
    q, k, v = normal(1, 1, 2, sq, 64), normal(2, 1, 2, 300, 64), normal(3, 1, 2, 300, 64)
    q[:, :, ::8] *= 1e7
    rules = dict(softcap=1e6, causal=False)
    got, (want, err) = attend(bridge, buffers, dtype, q, k, v, **rules), expected(dtype, q, k, v, **rules)
    assert np.isfinite(got).all()
    low = np.arange(sq) % 8 != 0
    within(got[:, :, low], want[:, :, low], err[:, :, low])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("sq", [1, 64, 200])
@pytest.mark.parametrize("softcap", [0.0, 30.0, 1e3])
@pytest.mark.parametrize("sk", [200, 1300])
def test_attention_does_not_see_what_a_cache_holds_behind_a_length(bridge, buffers, dtype, d, sq, softcap, sk):
    """Results are the same bit for bit whatever lies behind the length: zeros, large numbers, infinities or NaN."""
    lengths = [sk - 5, sk - 150, 1]
    q, k, v = normal(1, 3, 4, sq, d), normal(2, 3, 2, sk, d), normal(3, 3, 2, sk, d)
    got = []
    for behind in (0.0, 3e4, -np.inf, np.nan):
        for i, n in enumerate(lengths):
            k[i, :, n:], v[i, :, n:] = behind, behind
        got.append(attend(bridge, buffers, dtype, q, k, v, lengths=lengths, starts=[0, 3, 0], softcap=softcap, causal=sq > 64))
    for other in got[1:]:
        assert np.array_equal(got[0], other)


def refuse_for_long(bridge, buffers):
    """A call whose every CTA reports its length, waves of them one after another: 2048 sequences of one long cache."""
    b, h, sk, d = 2048, 8, 16384, 128
    q = buffers.put(np.zeros((b, h, 1, d), np.float32), "bfloat16")
    k = buffers.put(np.zeros((1, h, sk, d), np.float32), "bfloat16")
    n = buffers.put(np.full(b, sk + 1), "int32")
    view = HeadView(k, (0, d, sk * d))
    bridge.synchronize()
    return buffers.own(bridge.decoder_attention(q, view, view, b, h, h, 1, sk, d, "bfloat16", lengths=n))


@pytest.mark.parametrize("who", ["serving call", "plan"])
def test_a_refusal_in_flight_is_reported_once(bridge, buffers, who):
    """The refused call still runs, and still reports, when the next call learns of it; a valid call after that one succeeds."""
    x = normal(1, 1, 1, 256, 256)
    h = buffers.put(x, "float32")
    call = {"serving call": lambda: bridge.decoder_attention(h, h, h, 1, 1, 1, 256, 256, 256, "float32"),
            "plan": lambda: bridge.matmul(h, h, 256, 256, 256, "float32")}[who]
    for _ in range(3):
        refuse_for_long(bridge, buffers)
        with pytest.raises(KernelError) as e:
            while True:                                   # until the first report has crossed to the host
                buffers.own(call())
        assert e.value.status == 7
        got = buffers.get(buffers.own(call()), x.shape, "float32")
        assert np.isfinite(got).all() and np.abs(got).max() > 0
        bridge.synchronize()


def test_two_refused_calls_in_flight_leave_the_next_valid_one_alone(bridge, buffers):
    x = normal(1, 1, 2, 3, 64)
    h = buffers.put(x, "float32")
    n = buffers.put(np.array([4]), "int32")
    for _ in range(3):
        refuse_for_long(bridge, buffers)
        with pytest.raises(KernelError) as e:
            while True:
                buffers.own(bridge.decoder_attention(h, h, h, 1, 2, 2, 3, 3, 64, "float32", lengths=n))
        assert e.value.status == 7
        out = buffers.own(bridge.decoder_attention(h, h, h, 1, 2, 2, 3, 3, 64, "float32"))
        assert np.isfinite(buffers.get(out, x.shape, "float32")).all()


def test_a_small_call_of_another_thread_leaves_a_large_one_its_shared_memory(bridge, buffers):
    """One bridge moves from thread to thread, each call behind the one before it: the limit of a kernel's shared memory is the
    device's, not the thread's."""
    u = buffers.put(np.full(2, 0.5, np.float32), "float32")
    rows = {n: normal(n, 2, n) for n in (1000, 200003)}
    dev = {n: buffers.put(x, "float32") for n, x in rows.items()}
    keys = {n: buffers.put(normal(n, 1, 1, n, 128), "bfloat16") for n in (200, 40000)}
    q = buffers.put(normal(5, 1, 1, 100, 128), "bfloat16")

    def calls(vocab, sk):
        out = buffers.own(bridge.sample_tokens(dev[vocab], u, 2, vocab, "float32"))
        att = buffers.own(bridge.decoder_attention(q, keys[sk], keys[sk], 1, 1, 1, 100, sk, 128, "bfloat16"))
        return buffers.get(out, (2,), "int64"), buffers.get(att, (1, 1, 100, 128), "bfloat16")

    with ThreadPoolExecutor(1) as one, ThreadPoolExecutor(1) as two:
        first = one.submit(calls, 200003, 40000).result()
        small = two.submit(calls, 1000, 200).result()
        again = one.submit(calls, 200003, 40000).result()
        assert np.array_equal(two.submit(calls, 1000, 200).result()[1], small[1])
    for a, b in zip(first, again):
        assert np.array_equal(a, b)
    assert list(first[0]) == [oracle.sample(r, 0.5, np.float32(1.0))[0] for r in rows[200003]]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sq,group", [(1, 1), (1, 4), (4, 8), (64, 1), (130, 1)])
@pytest.mark.parametrize("at", [0, 70000, 131077])
def test_attention_keeps_what_many_small_probabilities_add_up_to(bridge, buffers, dtype, sq, group, at):
    """One key 18 above 131077 others: each of those has a probability of 2^-26, below what float16 holds beside a largest one
    of 1, and together they have 2^-9.  The largest key's value is zero, so that they are the whole result."""
    sk, d = 131078, 64
    q, k, v = np.zeros((1, group, sq, d), np.float32), np.zeros((1, 1, sk, d), np.float32), np.ones((1, 1, sk, d), np.float32)
    q[..., 0], k[:, :, at, 0], v[:, :, at] = 1.0, 18.0, 0.0
    rules = dict(scale=1.0, causal=False)
    want = np.full(q.shape, (sk - 1) / (sk - 1 + np.exp(18.0)))
    # scores are exact; a probability is rounded relatively (HALF), in float16 by at least half its smallest step, 2^-25 of a
    # reference that lies at most 2^7 below the largest; the sums over the keys (32 bits, n terms) and the exponential as in attention()
    err = want * (2 * oracle.HALF[dtype] + 2 * (sk * 2.0 ** -24 + 2.0 ** -21)) + (sk * 2.0 ** -32 if dtype == "float16" else 0.0)
    within(attend(bridge, buffers, dtype, q, k, v, **rules), want, err)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", [1, 4, 24])
def test_attention_keeps_small_probabilities_of_unsplit_caches(bridge, buffers, dtype, group):
    """The same for a batch so large that no sequence's keys are split over CTAs: the warps that do not meet the largest key have
    references of their own, the one that does holds a part of the others."""
    b, sk, d = 300, 16384, 64
    q, k, v = np.zeros((b, group, 1, d), np.float32), np.zeros((1, 1, sk, d), np.float32), np.ones((1, 1, sk, d), np.float32)
    q[..., 0], k[:, :, 0, 0], v[:, :, 0] = 1.0, 18.0, 0.0
    views = [HeadView(buffers.put(x, dtype), (0, d, sk * d)) for x in (k, v)]
    out = buffers.own(bridge.decoder_attention(buffers.put(q, dtype), *views, b, group, 1, 1, sk, d, dtype, scale=1.0, causal=False))
    want = np.full(q.shape, (sk - 1) / (sk - 1 + np.exp(18.0)))
    err = want * (2 * oracle.HALF[dtype] + 2 * (sk * 2.0 ** -24 + 2.0 ** -21)) + (sk * 2.0 ** -32 if dtype == "float16" else 0.0)
    within(buffers.get(out, q.shape, dtype), want, err)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("sq", [1, 64, 200])
@pytest.mark.parametrize("size,factor", [(3.0, 1.0), (300.0, 1.0), (6e4, 1.0), (6e4, 50.0), (6e4, 1e3), (6e4, 2e4), (6e4, 1e19)])
def test_attention_with_large_scores_stays_finite(bridge, buffers, dtype, d, sq, size, factor):
    """Scores from tens to 10^24 of either sign, which rise along the keys of one head and fall along the other's: no
    probability passes its type, and where 32 bits leave the exponents no digits the results are averages of values still."""
    sk = 700
    q, k, v = np.ones((1, 2, sq, d), np.float32), np.zeros((1, 2, sk, d), np.float32), normal(3, 1, 2, sk, d)
    k[..., 0] = np.linspace(-1, 1, sk) * size
    k[:, 1] = k[:, 1, ::-1]
    rules = dict(scale=8.0 * min(factor, 1e17), causal=False)
    q *= max(factor / 1e17, 1.0)
    got = attend(bridge, buffers, dtype, q, k, v, **rules)
    assert np.isfinite(got).all()
    if size < 1e3:
        within(got, *expected(dtype, q, k, v, **rules))
    else:
        top = np.abs(rounded(v, dtype)).max()
        assert np.abs(got).max() <= top * (1 + 2.0 ** -6) and np.abs(got).max(-1).min() > 1e-3


@pytest.mark.parametrize("vocab", [131072, 600011, 1 << 20])
def test_sampling_reaches_a_flat_tail(bridge, buffers, vocab):
    """One token above a tail that together has 2^-22.6 of its weight (2^-42.6 each for the largest vocabulary): the last number
    below one falls into the tail, and the token's interval of the exact running sum lies within 2^-24 of the number."""
    x = np.full((4, vocab), np.float32(np.log(2.0 ** -22.6 / vocab)), np.float32)
    top = [0, 0, vocab // 2, vocab - 1]
    x[np.arange(4), top] = 0.0
    u = np.float32([1 - 2.0 ** -24, 1 - 2.0 ** -23, 1 - 2.0 ** -24, 2.0 ** -24])
    got, _ = run_sample(bridge, buffers, x, u, "float32")
    for i in range(4):
        w = np.exp(x[i].astype(np.float64))
        sums, at = np.cumsum(w), int(got[i])
        # a weight is a whole number of 2^-43 of the largest or less: half a unit each, the same for equal ones
        slack = 2.0 ** -24 * sums[-1]
        assert 0 <= at < vocab
        assert sums[at] - w[at] - slack <= float(u[i]) * sums[-1] <= sums[at] + slack, (i, at)
    assert got[0] > 0


def test_sampling_refuses_a_vocabulary_its_sums_are_too_coarse_for(bridge, buffers):
    n = (1 << 20) + 1
    x, u = buffers.put(np.zeros((1, n), np.float32), "float32"), buffers.put(np.zeros(1, np.float32), "float32")
    with pytest.raises(KernelError) as e:
        buffers.own(bridge.sample_tokens(x, u, 1, n, "float32"))
    assert e.value.status == 2
    assert run_sample(bridge, buffers, np.zeros((1, n - 1), np.float32), np.float32([0.5]), "float32")[0][0] == (n - 1) // 2


@pytest.mark.parametrize("sq", [1, 64])
def test_a_device_side_refusal_names_its_operator(bridge, buffers, sq):
    x = buffers.put(normal(1, 1, 1, sq, 64), "bfloat16")
    caches = [buffers.put(normal(2, 1, 1, 80, 64), "bfloat16") for _ in range(2)]
    bad = buffers.put(np.array([81]), "int32")
    out = buffers.own(bridge.decoder_attention(x, *caches, 1, 1, 1, sq, 80, 64, "bfloat16", lengths=bad))
    with pytest.raises(KernelError, match="decoder_attention: a length outside the cache") as e:
        bridge.materialize(out, (1, 1, sq, 64), "bfloat16")
    assert e.value.status == 7
    out = buffers.own(bridge.rotary_append(x, x, x, *caches, RotarySpec(64), 1, 1, 1, sq, 80, 64, "bfloat16", starts=bad))
    with pytest.raises(KernelError, match="rotary_append: a count or a cache row outside its buffer") as e:
        bridge.synchronize()
    assert e.value.status == 7


@pytest.mark.parametrize("d", [32, 64])
@pytest.mark.parametrize("sq,sk", [(64, 512), (128, 448), (200, 512)])
def test_attention_of_float32_prompts_adds_without_a_bias(bridge, buffers, d, sq, sk):
    """Nearly equal scores over values of one sign: the result is a mean, to which every key adds.  An error e_j in the exponent
    of probability p_j moves it by p_j e_j (v_j - mean); e_j: the dot product as in attention(), scaling and exponential 2^-21.
    The rest is relative to the mean: the split of probabilities and of values drops 2^-21 each; the tensor core adds with
    truncation, a step of 2^-23 for each of a tile's 8 products of the upper parts and two more for the small ones; the tiles are
    added in 32 bits, half a step each, the probabilities by 18 such additions in a tile and one for each tile, and the division
    and its product are two halves more."""
    q, k = 0.05 * normal(4, 2, 2, sq, d), normal(6, 2, 2, sk, d)
    v = 3.0 + np.clip(normal(5, 2, 2, sk, d), -3, 3) / 4
    got = attend(bridge, buffers, "float32", q, k, v, causal=False)
    q, k, v = (x.astype(np.float64) for x in (q, k, v))
    p = np.exp(q @ k.swapaxes(-1, -2) / np.sqrt(d))
    p /= p.sum(-1, keepdims=True)
    want = p @ v
    p = p * ((d + 16) * 2.0 ** -23 * (np.abs(q) @ np.abs(k).swapaxes(-1, -2)) / np.sqrt(d) + 2.0 ** -21)
    err = p @ np.abs(v - 3.0) + p.sum(-1, keepdims=True) * np.abs(want - 3.0) + want * (2 * 2.0 ** -21 + 10 * 2.0 ** -23 + (2 * (sk // 64) + 18 + 2) * 2.0 ** -24)
    within(got, want, err)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("sq,rule", [(64, "plain"), (130, "plain"), (300, "ragged"), (64, "capped")])
def test_attention_of_long_caches_adds_without_a_bias(bridge, buffers, dtype, d, sq, rule):
    """Equal scores over 140000 values of one sign, whose mean is the result.  The tensor core adds with truncation: 16 keys at a
    time, two steps of 2^-23 each (of the products' sum and of the accumulator), for at most 64 tiles of 128 keys, 2^-13 of the
    mean in all; then come the half step of the result and a few of 32 bits.  Left to itself the sum loses 2^-10 of itself."""
    sk = 140000
    rules = dict(causal=False, softcap=30.0 if rule == "capped" else 0.0)
    if rule == "ragged":
        rules.update(lengths=[sk, 70001])
    v = 3.0 + np.clip(normal(5, 2, 1, sk, d), -3, 3) / 4
    got = attend(bridge, buffers, dtype, np.zeros((2, 2, sq, d), np.float32), normal(6, 2, 1, sk, d), v, **rules)
    v = rounded(v, dtype)
    want = np.stack([v[i, :, :n].mean(1) for i, n in enumerate(rules.get("lengths", [sk, sk]))])[:, :, None]
    want = np.broadcast_to(want, got.shape)
    within(got, want, want * (2.0 ** -13 + oracle.HALF[dtype] + 2.0 ** -20))


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rule", ["causal", "rising", "documents", "rows that begin late"])
def test_attention_of_prompts_over_long_caches(bridge, buffers, dtype, d, rule):
    """Sums that go on in memory: over references that rise on the way, rows that see their first key there, and few tiles."""
    b, sq, sk = 1, 140, 26000
    q, k, v = normal(1, b, 2, sq, d), normal(2, b, 1, sk, d), normal(3, b, 1, sk, d)
    rules = dict(starts=[sk - sq])
    if rule == "rising":
        q, k = np.abs(q), k * 0.1
        k[:, :, :, 0] = np.linspace(-8, 8, sk)
    if rule == "documents":
        rules.update(documents=np.repeat([0, 1], [9000, 17000])[None].astype(np.int32), starts=[9000 - sq // 2])
    if rule == "rows that begin late":
        ids = np.zeros((b, sk), np.int32)
        ids[:, 12000:] = 1
        rules.update(documents=ids, causal=False, starts=[12000 - sq // 2])
    got = attend(bridge, buffers, dtype, q, k, v, **rules)
    within(got, *expected(dtype, q, k, v, **rules))


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("d,group,sq", [(64, 8, 4), (128, 1, 1), (128, 8, 4), (128, 1, 63), (256, 1, 63)])
def test_attention_of_many_long_caches_adds_without_a_bias(bridge, buffers, dtype, d, group, sq):
    """The same where so many sequences fill the device that none is split for speed.  A group of warps adds at most 16384 keys
    (bfloat16 131072) in the tensor core, 16 at a time, two steps of 2^-23 each: 2^-12 of the mean, or 2^-9."""
    b, sk = 296, 500000
    q = np.zeros((b, group, sq, d), np.float32)
    k, v = normal(6, 1, 1, sk, d), 3.0 + np.clip(normal(5, 1, 1, sk, d), -3, 3) / 4
    views = [HeadView(buffers.put(x, dtype), (0, d, sk * d)) for x in (k, v)]
    out = buffers.own(bridge.decoder_attention(buffers.put(q, dtype), *views, b, group, 1, sq, sk, d, dtype, causal=False))
    want = np.broadcast_to(rounded(v, dtype).mean(2, keepdims=True), q.shape)
    within(buffers.get(out, q.shape, dtype), want, want * ((2.0 ** -12 if dtype == "float16" else 2.0 ** -9) + oracle.HALF[dtype] + 2.0 ** -20))
