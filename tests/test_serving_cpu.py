"""CPU: the serving operators' C structures and views as the header lays them out, refusals that need no device, and the
64-bit definitions the GPU tests compare against."""
import ctypes as C

import numpy as np
import pytest

from browsergrad_b200 import HeadView, RotarySpec, _lib
from browsergrad_b200.errors import KernelError
from tests import serving_oracle as oracle


def test_structures_match_the_header():
    assert C.sizeof(HeadView) == 8 + 8 + 3 * 8
    assert C.sizeof(RotarySpec) == 4 * 4 + 6 * 8
    assert C.sizeof(_lib.AttentionRules) == 2 * 8 + 2 * 4 + 5 * 8
    assert C.sizeof(_lib.Sampling) == 3 * 8 + 8 + 4 * 8


def test_views_address_what_they_say():
    b, rows, heads, dim = 2, 5, 3, 4
    flat = np.arange(b * rows * heads * dim)
    for make, array in ((HeadView.heads_first, flat.reshape(b, heads, rows, dim).transpose(0, 2, 1, 3)),
                        (HeadView.rows_first, flat.reshape(b, rows, heads, dim))):
        v = make(7, rows, heads, dim)
        assert v.handle == 7
        for i in range(b):
            for s in range(rows):
                for h in range(heads):
                    at = v.offset + i * v.stride[0] + s * v.stride[1] + h * v.stride[2]
                    assert (flat[at:at + dim] == array[i, s, h]).all()
    packed = HeadView.rows_first(7, rows, heads, dim, first=2)
    assert packed.offset == 2 * dim and list(packed.stride) == [rows * heads * dim, heads * dim, dim]


def test_an_unknown_scaling_is_refused():
    with pytest.raises(KernelError):
        RotarySpec(64, scaling="cubic")
    assert RotarySpec(64, scaling="ramp", factor=8.0, original_length=4096).scaling == 2


def test_null_arguments_are_refused_without_a_device():
    lib, out = _lib.load(), C.c_int64()
    v, spec, rules, sampling = HeadView(1, (1, 1, 1)), RotarySpec(2), _lib.AttentionRules(), _lib.Sampling()
    r = C.byref(out)
    assert lib.bg_rotary(None, v, spec, 1, 1, 1, 2, 1, 0, 0, 0, None, r) == 1
    assert lib.bg_rotary_append(None, v, v, v, v, v, spec, 1, 1, 1, 1, 1, 2, 1, 0, 0, 0, None, r) == 1
    assert lib.bg_decoder_attention(None, v, v, v, 1, 1, 1, 1, 1, 2, 1, rules, None, r) == 1
    assert lib.bg_sample_tokens(None, 1, 1, 1, 1, 1, sampling, 0, 0, r) == 1


def test_rotary_definition_turns_pairs():
    """Each pair keeps its length, turning back undoes turning, and the gradient of sum(g * turned) is g turned back."""
    rng = np.random.default_rng(0)
    x, g = rng.standard_normal((2, 1, 3, 2, 8))
    pos, f = np.array([[0, 1, 50]]), oracle.frequencies(8)
    for inter in (False, True):
        y, _ = oracle.rotary(x, pos, f, inter)
        assert np.allclose((y ** 2).sum(-1), (x ** 2).sum(-1)) and np.allclose(y[:, 0], x[:, 0])
        assert np.allclose(oracle.rotary(y, pos, f, inter, inverse=True)[0], x)
        grad, _ = oracle.rotary(g, pos, f, inter, inverse=True)
        i, eps = (0, 2, 1, 5), 1e-6
        bumped = x.copy()
        bumped[i] += eps
        assert np.isclose(((oracle.rotary(bumped, pos, f, inter)[0] - y) * g).sum() / eps, grad[i], atol=1e-6)


def test_visibility_definition():
    seen, pos = oracle.visible(2, 3, 6, True, lengths=[6, 4], prefixes=[0, 2])
    assert pos.tolist() == [[3, 4, 5], [1, 2, 3]]
    assert seen[0].sum(-1).tolist() == [4, 5, 6] and seen[1].sum(-1).tolist() == [2, 3, 4]
    docs = np.array([[0, 0, 1, 1, -1, 1]])
    seen, _ = oracle.visible(1, 6, 6, True, documents=docs)
    assert seen[0].sum(-1).tolist() == [1, 2, 1, 2, 0, 3]


def test_sampling_definition():
    x = np.array([1.0, 3.0, 3.0, 2.0], np.float32)
    assert oracle.sample(x, 0.9, np.float32(0.0)) == (1, 1.0)
    assert oracle.sample(x, 0.999, np.float32(1.0), top_k=2)[0] == 2
    assert oracle.sample(x, 0.999, np.float32(1.0), top_k=1)[0] == 1
    assert oracle.sample(x, 0.5, np.float32(1.0), top_p=0.3) == (1, 1.0)
    assert oracle.sample(np.full(3, -np.inf, np.float32), 0.5, np.float32(1.0)) == (-1, 0.0)
    p = np.exp(x - 3.0) / np.exp(x - 3.0).sum()
    for u in np.linspace(0, 0.99, 34):
        assert oracle.sample(x, u, np.float32(1.0))[0] == int(np.searchsorted(np.cumsum(p), np.float32(u), side="right"))
