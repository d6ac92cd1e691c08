"""The operators of a decoder's serving loop, measured case by case: rotary positions (alone, and fused with the append
to a key / value cache), attention over such a cache with scores that are capped, biased by distance or masked by rule,
and the choice of the next token from the logits.

``run`` computes a case in elementary torch operations (``own`` false) or through ``CudaBridge`` (``own`` true); ``exact``
states the same operator in 64 bits.
"""
import math
import random

import numpy as np
import torch

own = False

_TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def listed():
    """Sizes: 12 heads of 64, a vocabulary of 32000, prompts of 1024 and 2048 and a batch of 8 are the benchmark's
    decoder; grouped heads of 128, longer caches and a vocabulary of 128000 are the usual larger ones."""
    return [
        # One generated token for a batch of 8 in the benchmark's decoder: latency of the smallest append.
        _rotary("append one token", form="append", dtype="bfloat16", b=8, s=1, hq=12, hkv=12, d=64, rot=64, cap=1024),
        # A ragged batch of prompts entering the cache, interleaved pairs on half of the head (odd token count).
        _rotary("append prompts, interleaved", form="append", dtype="float16", b=6, s=1537, hq=32, hkv=8, d=128, rot=64,
                interleaved=True, cap=2048, ragged=True),
        # The benchmark decoder's fp32 prompts, every dimension rotated.
        _rotary("rotate fp32", form="rotate", dtype="float32", b=8, s=1024, hq=12, hkv=0, d=64, rot=64),
        # One long document far behind position zero, frequencies stretched by wavelength.
        _rotary("rotate far positions", form="rotate", dtype="bfloat16", b=1, s=32771, hq=32, hkv=0, d=128, rot=128,
                start=900001, scaling="ramp", factor=8.0, original=8192),
        # One generated token over short caches of the benchmark's decoder: latency of a decode step.
        _attention("decode, short caches", dtype="bfloat16", b=8, hq=12, hkv=12, sq=1, sk=1024, d=64, ragged=True),
        # One generated token, grouped heads, ragged lengths, capped scores: a full serving batch.
        _attention("decode, capped", dtype="bfloat16", b=32, hq=32, hkv=8, sq=1, sk=8192, d=128, cap=50.0, ragged=True),
        # One sequence with a very long cache and a bias by distance, four tokens checked at once.
        _attention("decode, one long cache", dtype="float16", b=1, hq=32, hkv=4, sq=4, sk=131077, d=128, alibi=True),
        # Packed documents of the benchmark's attention length.
        _attention("prompt, packed documents", dtype="bfloat16", b=4, hq=12, hkv=12, sq=2048, sk=2048, d=64, docs=5),
        # A prompt whose first part is seen by everyone, capped, grouped heads.
        _attention("prompt, prefix and cap", dtype="float16", b=2, hq=16, hkv=4, sq=4099, sk=4099, d=128, cap=30.0,
                   prefix=700),
        # The fp32 decoder with a bias by distance and padded prompts.
        _attention("prompt, fp32 biased", dtype="float32", b=8, hq=12, hkv=12, sq=1024, sk=1024, d=64, alibi=True,
                   ragged=True),
        # The benchmark's vocabulary, a small batch with every filter.
        _sample("sample, small batch", dtype="float32", n=8, vocab=32000, top_k=50, top_p=0.9, min_p=0.02),
        # A large vocabulary and a large batch, nucleus only.
        _sample("sample, large vocabulary", dtype="bfloat16", n=200, vocab=128001, top_k=0, top_p=0.95, min_p=0.0),
    ]


def _rotary(name, form, dtype, b, s, hq, hkv, d, rot, interleaved=False, cap=0, ragged=False, start=0, scaling="none",
            factor=1.0, original=0, base=10000.0):
    return dict(name=name, op="rotary", form=form, dtype=dtype, b=b, s=s, hq=hq, hkv=hkv, d=d, rot=rot,
                interleaved=interleaved, cap=cap, ragged=ragged, start=start, scaling=scaling, factor=factor,
                original=original, base=base)


def _attention(name, dtype, b, hq, hkv, sq, sk, d, cap=0.0, alibi=False, docs=0, prefix=0, ragged=False, causal=True):
    return dict(name=name, op="attention", dtype=dtype, b=b, hq=hq, hkv=hkv, sq=sq, sk=sk, d=d, cap=cap, alibi=alibi,
                docs=docs, prefix=prefix, ragged=ragged, causal=causal)


def _sample(name, dtype, n, vocab, top_k, top_p, min_p):
    return dict(name=name, op="sample", dtype=dtype, n=n, vocab=vocab, top_k=top_k, top_p=top_p, min_p=min_p)


def _spread(rng, low, high):
    """A whole number between the two, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("rotate", "append", "decode", "prompt", "sample"))
    if kind in ("rotate", "append"):
        d = rng.choice((64, 80, 128))
        hkv = rng.choice((1, 4, 8, 12))
        hq = hkv * rng.choice((1, 2, 4))
        s = _spread(rng, 1, 4096)
        b = max(1, min(_spread(rng, 1, 64), 4_000_000 // (s * hq * 2 + hkv * d)))
        scaling = rng.choice(("none", "linear", "ramp"))
        case = _rotary("", form=kind, dtype=rng.choice(sorted(_TYPES)), b=b, s=s, hq=hq, hkv=hkv, d=d,
                       rot=rng.choice((d, d // 2)), interleaved=rng.random() < 0.5, cap=s + _spread(rng, 1, 2048),
                       ragged=rng.random() < 0.5, start=rng.randrange(100000) if kind == "rotate" else 0,
                       scaling=scaling, factor=1.0 if scaling == "none" else rng.choice((2.0, 4.0, 8.0)),
                       original=4096 if scaling == "ramp" else 0, base=rng.choice((10000.0, 500000.0)))
        if kind == "rotate":
            case.update(hkv=0, cap=0, ragged=False)
    elif kind == "decode":
        hkv = rng.choice((1, 2, 4, 8, 12))
        group = rng.choice((1, 2, 4, 8))
        sq = rng.choice((1, 1, 1, 2, 5))
        sk = _spread(rng, 16, 60000)
        d = rng.choice((64, 96, 128))
        dtype = rng.choice(sorted(_TYPES))
        b = max(1, min(_spread(rng, 1, 64), (90_000_000 if dtype == "float32" else 180_000_000) // (hkv * sk * d),
                       60_000_000 // (hkv * group * sq * sk)))
        case = _attention("", dtype=dtype, b=b, hq=hkv * group, hkv=hkv, sq=min(sq, sk), sk=sk, d=d,
                          cap=rng.choice((0.0, 30.0, 50.0)), alibi=rng.random() < 0.4, ragged=rng.random() < 0.6)
    elif kind == "prompt":
        hkv = rng.choice((1, 2, 4, 12))
        group = rng.choice((1, 2, 4))
        s = _spread(rng, 64, 4100)
        b = max(1, min(_spread(rng, 1, 16), 300_000_000 // (hkv * group * s * s)))
        rule = rng.choice(("plain", "docs", "prefix", "both ways"))
        case = _attention("", dtype=rng.choice(("float16", "bfloat16", "bfloat16", "float32")), b=b, hq=hkv * group, hkv=hkv,
                          sq=s, sk=s, d=rng.choice((64, 64, 80, 128)), cap=rng.choice((0.0, 0.0, 30.0, 50.0)),
                          alibi=rng.random() < 0.4, docs=rng.randrange(2, 9) if rule == "docs" else 0,
                          prefix=rng.randrange(1, s) if rule == "prefix" else 0, ragged=rng.random() < 0.4,
                          causal=rule != "both ways")
    else:
        vocab = _spread(rng, 1000, 200000)
        case = _sample("", dtype=rng.choice(sorted(_TYPES)), n=max(1, min(_spread(rng, 1, 256), 25_000_000 // vocab)),
                       vocab=vocab, top_k=rng.choice((0, 1, 20, 50, 400)), top_p=rng.choice((1.0, 0.95, 0.8)),
                       min_p=rng.choice((0.0, 0.02, 0.1)))
    del case["name"]
    return case


# -- what a case's whole-number inputs are: the same for every seed, so that work() can count by them -------------------


def _lengths(case):
    """Valid keys of each sequence (attention), or new tokens of each (append)."""
    full = case["sk"] if case["op"] == "attention" else case["s"]
    if not case["ragged"]:
        return [full] * case["b"]
    low = case["sq"] if case["op"] == "attention" and case["sq"] < case["sk"] else 1
    rng = random.Random(full * 31 + case["b"])
    got = [rng.randint(max(low, full // 4), full) for _ in range(case["b"])]
    got[rng.randrange(case["b"])] = full
    return got


def _first_rows(case):
    """Cache row of each sequence's first new token (append)."""
    rng = random.Random(case["cap"] * 17 + case["b"])
    return [rng.randint(0, case["cap"] - case["s"]) for _ in range(case["b"])]


def _starts(case):
    """Position of the first query row: prompts begin at zero, generated tokens are the last ones of their sequence."""
    return [0 if case["sq"] == case["sk"] else n - case["sq"] for n in _lengths(case)]


def _document_ends(case):
    """Ends of the packed documents; the last tokens of the buffer belong to none."""
    n, s = case["docs"], case["sk"]
    used = s - s // 50
    return [max(i + 1, int(used * ((i + 1) / n) ** 1.3)) for i in range(n)]


def _documents(case):
    ids = np.full(case["sk"], -1, np.int32)
    begin = 0
    for i, end in enumerate(_document_ends(case)):
        ids[begin:end] = i
        begin = max(begin, end)
    return np.tile(ids, (case["b"], 1))


def _visible_pairs(case):
    """Pairs of a query row and a key that see each other, over the batch, for one head."""
    total = 0
    for start, length in zip(_starts(case), _lengths(case)):
        pos = np.arange(start, start + case["sq"], dtype=np.int64)
        if not case["causal"]:
            first, last = np.zeros_like(pos), np.full_like(pos, length)
        else:
            first = np.zeros_like(pos)
            last = np.minimum(np.maximum(pos + 1, case["prefix"]), length)
            last[pos >= length] = 0
        if case["docs"]:
            ends = np.asarray(_document_ends(case))
            which = np.searchsorted(ends, pos, side="right")
            begins = np.concatenate([[0], ends])
            inside = which < len(ends)
            first = np.where(inside, begins[which], 0)
            last = np.where(inside, np.minimum(last, np.concatenate([ends, [0]])[which]), 0)
        total += int(np.maximum(last - first, 0).sum())
    return total


def work(case):
    es = torch.empty((), dtype=_TYPES[case["dtype"]]).element_size()
    if case["op"] == "rotary":
        tokens = case["b"] * case["s"]
        moved = 2 * tokens * case["hq"] * case["d"]
        pairs = tokens * case["hq"] * case["rot"] // 2
        if case["form"] == "append":
            new = sum(_lengths(case))
            moved += 4 * new * case["hkv"] * case["d"]
            pairs += new * case["hkv"] * case["rot"] // 2
        return {"bytes": moved * es, "flops": 6 * pairs}
    if case["op"] == "attention":
        keys = sum(_lengths(case))
        rows = case["b"] * case["sq"]
        return {"bytes": es * case["d"] * (2 * rows * case["hq"] + 2 * keys * case["hkv"]),
                "flops": 4 * case["d"] * case["hq"] * _visible_pairs(case)}
    return {"bytes": case["n"] * (case["vocab"] * es + 32), "flops": 8 * case["n"] * case["vocab"]}


# -- inputs -------------------------------------------------------------------------------------------------------------


def _tensors(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    t = _TYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(t)

    def whole(values):
        return torch.as_tensor(np.asarray(values, dtype=np.int32), device="cuda")

    b, st = case.get("b"), {}
    if case["op"] == "rotary":
        if case["form"] == "rotate":
            st["x"] = normal(b, case["s"], case["hq"], case["d"])
        else:  # one projection leaves q, k and v side by side
            st["qkv"] = normal(b, case["s"], case["hq"] + 2 * case["hkv"], case["d"])
            st["k_cache"] = normal(b, case["hkv"], case["cap"], case["d"])
            st["v_cache"] = normal(b, case["hkv"], case["cap"], case["d"])
            st["starts"] = whole(_first_rows(case))
            st["counts"] = whole(_lengths(case))
    elif case["op"] == "attention":
        st["q"] = normal(b, case["sq"], case["hq"], case["d"], scale=1.5)
        if case["sq"] == case["sk"]:  # a prompt: keys and values as the projections leave them
            st["k"] = normal(b, case["sk"], case["hkv"], case["d"])
            st["v"] = normal(b, case["sk"], case["hkv"], case["d"])
        else:
            st["k"] = normal(b, case["hkv"], case["sk"], case["d"])
            st["v"] = normal(b, case["hkv"], case["sk"], case["d"])
        st["lengths"] = whole(_lengths(case))
        st["starts"] = whole(_starts(case))
        if case["alibi"]:
            st["slopes"] = torch.as_tensor(_slopes(case), device="cuda")
        if case["docs"]:
            st["documents"] = whole(_documents(case))
        if case["prefix"]:
            st["prefixes"] = whole([case["prefix"]] * b)
    else:
        n = case["n"]
        # a few likely tokens over a broad background, as a trained head gives them
        x = torch.randn(n, case["vocab"], generator=g, device="cuda") * 1.8
        lift = torch.rand(n, case["vocab"], generator=g, device="cuda")
        x += torch.where(lift > 0.9995, 9.0 * torch.rand(n, case["vocab"], generator=g, device="cuda"), 0.0)
        st["logits"] = x.to(t)
        st["uniforms"] = torch.rand(n, generator=g, device="cuda")
        st["temperatures"] = 0.6 + 0.6 * torch.rand(n, generator=g, device="cuda")
        st["temperatures"][5::8] = 0.0  # some requests are greedy
    return st


def _slopes(case):
    return np.exp2(-8.0 * (np.arange(case["hq"]) + 1) / case["hq"]).astype(np.float32)


def prepare(case, seed):
    st = {"case": case, "in": _tensors(case, seed)}
    if own:
        st["own"] = _Device(case, st["in"])
        st["in"] = None
    return st


def run(st):
    if own:
        return st["own"].run()
    return {"rotary": _plain_rotary, "attention": _plain_attention, "sample": _plain_sample}[st["case"]["op"]](st["case"], st["in"])


# -- the framework's calls ----------------------------------------------------------------------------------------------

_BRIDGE = None


def _bridge():
    global _BRIDGE
    if _BRIDGE is None:
        from browsergrad_b200 import CudaBridge
        _BRIDGE = CudaBridge(0)
    return _BRIDGE


class _Buffer:
    """A device buffer of the bridge, as torch sees it; it lives as long as the tensors made of it."""

    _KIND = {"float32": "<f4", "float16": "<f2", "bfloat16": "<i2", "int32": "<i4", "int64": "<i8"}

    def __init__(self, shape, dtype):
        self.bridge, self.dtype = _bridge(), dtype
        self.handle = self.bridge.alloc(shape, dtype)
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": self._KIND[dtype], "version": 3,
                                         "data": (self.bridge.device_pointer(self.handle), False)}

    def tensor(self):
        t = torch.as_tensor(self, device="cuda")
        return t.view(torch.bfloat16) if self.dtype == "bfloat16" else t

    def __del__(self):
        self.bridge.release(self.handle)


class _Device:
    """A case's inputs and outputs in buffers of the bridge, and the call on them."""

    def __init__(self, case, tensors):
        self.bridge, self.case = _bridge(), case
        buffers = {k: _Buffer(tuple(v.shape), str(v.dtype).replace("torch.", "")) for k, v in tensors.items()}
        self.h, self.views = {k: v.handle for k, v in buffers.items()}, {k: v.tensor() for k, v in buffers.items()}
        getattr(self, "_setup_" + case["op"])()
        self.bridge.synchronize()  # the buffers are there
        for k, v in tensors.items():
            self.views[k].copy_(v)
        torch.cuda.synchronize()

    def _new(self, shape, dtype):
        buffer = _Buffer(shape, dtype)
        return buffer.handle, buffer.tensor()

    def _setup_rotary(self):
        from browsergrad_b200 import HeadView, RotarySpec
        c, h = self.case, self.h
        self.spec = RotarySpec(c["rot"], base=c["base"], interleaved=c["interleaved"], scaling=c["scaling"],
                               factor=c["factor"], low=1.0, high=4.0, original_length=c["original"])
        out, self.out = self._new((c["b"], c["s"], c["hq"], c["d"]), c["dtype"])
        self.out_view = HeadView.rows_first(out, c["s"], c["hq"], c["d"])
        if c["form"] == "rotate":
            self.x = HeadView.rows_first(h["x"], c["s"], c["hq"], c["d"])
            return
        packed = c["hq"] + 2 * c["hkv"]
        self.q, self.k, self.v = (HeadView.rows_first(h["qkv"], c["s"], packed, c["d"], first=first)
                                  for first in (0, c["hq"], c["hq"] + c["hkv"]))

    def _run_rotary(self):
        c, h = self.case, self.h
        if c["form"] == "rotate":
            self.bridge.rotary(self.x, self.spec, c["b"], c["hq"], c["s"], c["d"], c["dtype"], start=c["start"], out=self.out_view)
            return self.out
        self.bridge.rotary_append(self.q, self.k, self.v, h["k_cache"], h["v_cache"], self.spec, c["b"], c["hq"], c["hkv"],
                                  c["s"], c["cap"], c["d"], c["dtype"], starts=h["starts"], counts=h["counts"], out=self.out_view)
        return self.out, self.views["k_cache"], self.views["v_cache"]

    def _setup_attention(self):
        from browsergrad_b200 import HeadView
        c, h = self.case, self.h
        out, self.out = self._new((c["b"], c["sq"], c["hq"], c["d"]), c["dtype"])
        self.out_view = HeadView.rows_first(out, c["sq"], c["hq"], c["d"])
        self.q = HeadView.rows_first(h["q"], c["sq"], c["hq"], c["d"])
        make = HeadView.rows_first if c["sq"] == c["sk"] else HeadView.heads_first
        self.k, self.v = (make(h[x], c["sk"], c["hkv"], c["d"]) for x in "kv")

    def _run_attention(self):
        c, h = self.case, self.h
        self.bridge.decoder_attention(self.q, self.k, self.v, c["b"], c["hq"], c["hkv"], c["sq"], c["sk"], c["d"], c["dtype"],
                                      causal=c["causal"], softcap=c["cap"], slopes=h.get("slopes"), documents=h.get("documents"),
                                      prefixes=h.get("prefixes"), lengths=h["lengths"], starts=h["starts"], out=self.out_view)
        return self.out

    def _setup_sample(self):
        n = self.case["n"]
        self.tokens_handle, self.tokens = self._new((n,), "int64")
        self.prob_handle, self.prob = self._new((n,), "float32")

    def _run_sample(self):
        c, h = self.case, self.h
        self.bridge.sample_tokens(h["logits"], h["uniforms"], c["n"], c["vocab"], c["dtype"], temperatures=h["temperatures"],
                                  top_k=c["top_k"], top_p=c["top_p"], min_p=c["min_p"], out=self.tokens_handle,
                                  probabilities=self.prob_handle)
        return self.tokens, self.prob

    def run(self):
        return getattr(self, "_run_" + self.case["op"])()


# -- plain forms --------------------------------------------------------------------------------------------------------


def _frequencies(case):
    """Radians per position of each pair, in 64 bits."""
    j = torch.arange(case["rot"] // 2, dtype=torch.float64, device="cuda")
    f = torch.exp(j * (-2.0 * math.log(case["base"]) / case["rot"]))
    if case["scaling"] == "linear":
        f = f / case["factor"]
    elif case["scaling"] == "ramp":  # wavelengths that fit the trained length often stay, rare ones are stretched
        turns = f * (case["original"] / (2.0 * math.pi))
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0.0, 1.0)
        f = f * (keep + (1.0 - keep) / case["factor"])
    return f


def _rotated(case, x, positions):
    """x [B, S, H, D] at positions [B, S] (or [1, S])."""
    angle = positions.double()[..., None] * _frequencies(case)
    c, s = torch.cos(angle).float()[:, :, None, :], torch.sin(angle).float()[:, :, None, :]
    r = case["rot"]
    turned, rest = x[..., :r].float(), x[..., r:]
    if case["interleaved"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * c - b * s, a * s + b * c), dim=-1).flatten(-2)
    else:
        a, b = turned[..., : r // 2], turned[..., r // 2:]
        turned = torch.cat((a * c - b * s, a * s + b * c), dim=-1)
    return torch.cat((turned.to(x.dtype), rest), dim=-1)


def _plain_rotary(case, st):
    row = torch.arange(case["s"], device="cuda")[None, :]
    if case["form"] == "rotate":
        return _rotated(case, st["x"], row + case["start"])
    hq, hkv = case["hq"], case["hkv"]
    positions = row + st["starts"][:, None]
    q = _rotated(case, st["qkv"][:, :, :hq], positions)
    k = _rotated(case, st["qkv"][:, :, hq: hq + hkv], positions)
    v = st["qkv"][:, :, hq + hkv:]
    new = (row < st["counts"][:, None])[:, :, None, None]
    at = torch.arange(case["b"], device="cuda")[:, None], slice(None), positions
    st["k_cache"][at] = torch.where(new, k, st["k_cache"][at])  # rows behind the last new token stay as they were
    st["v_cache"][at] = torch.where(new, v, st["v_cache"][at])
    return q, st["k_cache"], st["v_cache"]


def _heads_first(case, x):
    return x.transpose(1, 2) if case["sq"] == case["sk"] else x


def _plain_attention(case, st):
    b, hq, hkv, sq, sk, d = (case[x] for x in ("b", "hq", "hkv", "sq", "sk", "d"))
    key = torch.arange(sk, device="cuda")
    there = key[None, :] < st["lengths"][:, None]
    q = st["q"].transpose(1, 2).float().reshape(b, hkv, hq // hkv * sq, d)
    k = _heads_first(case, st["k"]).float()
    v = torch.where(there[:, None, :, None], _heads_first(case, st["v"]).float(), 0.0)
    s = (torch.matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(d))).reshape(b, hq, sq, sk)
    if case["cap"]:
        s = case["cap"] * torch.tanh(s / case["cap"])
    pos = st["starts"][:, None] + torch.arange(sq, device="cuda")[None, :]
    if case["alibi"]:
        s = s - st["slopes"][None, :, None, None] * (pos[:, :, None] - key).abs().float()[:, None]
    seen = there[:, None, :].expand(b, sq, sk)
    if case["causal"]:
        below = key <= pos[:, :, None]
        if case["prefix"]:
            below = below | (key < st["prefixes"][:, None, None])
        seen = seen & below & ((pos >= 0) & (pos < st["lengths"][:, None]))[:, :, None]
    if case["docs"]:
        inside = (pos >= 0) & (pos < sk)
        mine = torch.where(inside, st["documents"].gather(1, pos.clamp(0, sk - 1).long()), -1)
        seen = seen & (mine[:, :, None] == st["documents"][:, None, :]) & (mine >= 0)[:, :, None]
    seen = seen[:, None]
    top = torch.where(seen, s, -torch.inf).amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(s - torch.where(top == -torch.inf, 0.0, top)), 0.0)
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0.0, 1.0, total)
    o = torch.matmul(p.reshape(b, hkv, hq // hkv * sq, sk), v).reshape(b, hq, sq, d)
    return o.transpose(1, 2).to(st["q"].dtype).contiguous()


def _plain_sample(case, st):
    x = st["logits"].double()
    t = st["temperatures"].double()[:, None]
    greedy = t <= 0.0
    top = x.amax(-1, keepdim=True)
    w = torch.where(x == -torch.inf, 0.0, torch.exp((x - top) / torch.where(greedy, 1.0, t)))
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    keep = torch.ones_like(ws, dtype=torch.bool)
    if case["top_k"]:
        keep[:, case["top_k"]:] = False
    if case["top_p"] < 1.0:
        within = torch.where(keep, ws, 0.0)
        before = torch.cat((torch.zeros_like(t), within.cumsum(-1)[:, :-1]), dim=-1)
        keep &= before < float(np.float32(case["top_p"])) * within.sum(-1, keepdim=True)
    keep &= ws >= float(np.float32(case["min_p"]))
    keep[:, 0] = True
    kept = torch.where(torch.zeros_like(keep).scatter(1, order, keep), w, 0.0)
    total = kept.cumsum(-1)
    last = (kept > 0.0).long().mul(torch.arange(case["vocab"], device="cuda")).amax(-1, keepdim=True)
    token = (total <= st["uniforms"].double()[:, None] * total[:, -1:]).sum(-1, keepdim=True)
    token = torch.where(greedy, order[:, :1], torch.minimum(token, last))
    chance = torch.where(greedy, 1.0, kept.gather(1, token) / total[:, -1:])
    return token[:, 0], chance[:, 0].float()


# -- the same in 64 bits ------------------------------------------------------------------------------------------------


def exact(case, seed):
    st = _tensors(case, seed)
    return {"rotary": _exact_rotary, "attention": _exact_attention, "sample": _exact_sample}[case["op"]](case, st)


def _exact_turn(case, x, positions):
    """Each pair of x [S, H, D] as a complex number, turned by its angle."""
    j = np.arange(case["rot"] // 2)
    f = np.power(np.float64(case["base"]), -2.0 * j / case["rot"])
    if case["scaling"] == "linear":
        f = f / case["factor"]
    if case["scaling"] == "ramp":
        share = np.clip((case["original"] * f / (2 * np.pi) - 1.0) / 3.0, 0.0, 1.0)
        f = (1.0 - share) * f / case["factor"] + share * f
    turn = torch.polar(torch.ones(len(positions), len(j), dtype=torch.float64),
                       torch.as_tensor(np.multiply.outer(np.asarray(positions, np.float64), f))).to(x.device)[:, None, :]
    y, half = x.double().clone(), case["rot"] // 2
    one, two = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if case["interleaved"] else (slice(0, half), slice(half, 2 * half))
    z = torch.complex(y[..., one].contiguous(), y[..., two].contiguous()) * turn
    y[..., one], y[..., two] = z.real, z.imag
    return y


def _exact_rotary(case, st):
    if case["form"] == "rotate":
        at = np.arange(case["s"]) + case["start"]
        return torch.stack([_exact_turn(case, x, at) for x in st["x"]])
    hq, hkv = case["hq"], case["hkv"]
    k, v, q = st["k_cache"].double(), st["v_cache"].double(), []
    for i, (first, count) in enumerate(zip(_first_rows(case), _lengths(case))):
        turned = _exact_turn(case, st["qkv"][i, :, : hq + hkv], np.arange(case["s"]) + first)
        q.append(turned[:, :hq])
        k[i, :, first: first + count] = turned[:count, hq:].transpose(0, 1)
        v[i, :, first: first + count] = st["qkv"][i, :count, hq + hkv:].double().transpose(0, 1)
    return torch.stack(q), k, v


def _exact_attention(case, st):
    sq, group = case["sq"], case["hq"] // case["hkv"]
    out = torch.zeros(case["b"], sq, case["hq"], case["d"], dtype=torch.float64, device="cuda")
    ids = torch.as_tensor(_documents(case)[0], device="cuda") if case["docs"] else None
    for i, (start, n) in enumerate(zip(_starts(case), _lengths(case))):
        rows = torch.arange(sq, device="cuda") + start
        keys = torch.arange(n, device="cuda")
        gap = rows[:, None] - keys[None, :]
        hidden = torch.zeros_like(gap, dtype=torch.bool)
        if case["causal"]:
            hidden = (gap < 0) & ~(keys < case["prefix"])[None, :]
            hidden |= (rows >= n)[:, None]
        if ids is not None:
            hidden |= (ids[rows][:, None] != ids[:n][None, :]) | (ids[rows] < 0)[:, None]
        empty = hidden.all(-1)
        for h in range(case["hq"]):
            g = h // group
            k, v = (_heads_first(case, st[x])[i, g, :n].double() for x in "kv")
            s = st["q"][i, :, h].double() @ k.T / math.sqrt(case["d"])
            if case["cap"]:
                s = torch.tanh(s / case["cap"]) * case["cap"]
            if case["alibi"]:
                s -= float(_slopes(case)[h]) * gap.abs()
            s.masked_fill_(hidden, -torch.inf)
            o = torch.softmax(s, -1) @ v
            out[i, :, h] = torch.where(empty[:, None], 0.0, o)
    return out


def _exact_sample(case, st):
    x = st["logits"].double().cpu().numpy()
    tokens, chances = [], []
    for row, u, t in zip(x, st["uniforms"].cpu().numpy().astype(np.float64), st["temperatures"].cpu().numpy().astype(np.float64)):
        order = np.argsort(-row, kind="stable")
        if t <= 0:
            tokens.append(order[0])
            chances.append(1.0)
            continue
        w = np.exp((row[order] - row[order[0]]) / t)
        n = min(case["top_k"] or len(w), len(w))
        if case["top_p"] < 1:
            sums = np.cumsum(w[:n])
            n = 1 + int(np.count_nonzero(sums[:-1] < float(np.float32(case["top_p"])) * sums[-1]))
        n = max(1, min(n, int(np.count_nonzero(w >= float(np.float32(case["min_p"]))))))
        chosen = np.sort(order[:n])
        weight = np.exp((row[chosen] - row[order[0]]) / t)
        sums = np.cumsum(weight)
        pick = min(int(np.searchsorted(sums, u * sums[-1], side="right")), n - 1)
        tokens.append(chosen[pick])
        chances.append(weight[pick] / sums[-1])
    return torch.as_tensor(np.asarray(tokens, np.int64)), torch.as_tensor(np.asarray(chances, np.float64))
