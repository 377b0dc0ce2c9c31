"""Host side of the attention operators: frequencies, fixed-point turns, argument checks of the C entry points, the
index arithmetic of a batch, and the 64-bit forms against closed forms. No GPU."""
import ctypes
import math

import pytest
import torch

from eva_b200 import _lib
from eva_b200 import attention as T
from oracle import attention as A


def test_frequencies():
    f, m = T.rotary_frequencies(64)
    assert m == 1.0 and f[0] == 1.0 and f[31] == pytest.approx(10000.0 ** (-62 / 64), rel=1e-15)
    assert T.rotary_frequencies(64, scaling="linear", factor=4.0)[0][3] == f[3] / 4
    ntk = T.rotary_frequencies(64, scaling="ntk", factor=8.0)[0]
    assert ntk[0] == 1.0 and ntk[31] == pytest.approx(f[31] / 8, rel=1e-12)   # the slowest pair is slowed by the factor


def test_yarn_frequencies():
    """Pairs that turn more than beta_fast times in the original length keep their frequency, those under beta_slow are divided."""
    f, _ = T.rotary_frequencies(64)
    y, m = T.rotary_frequencies(64, scaling="yarn", factor=40.0, original_len=4096)
    assert m == pytest.approx(0.1 * math.log(40) + 1)
    for a, b in zip(f, y):
        turns = 4096 * a / (2 * math.pi)
        assert a / 40 * (1 - 1e-12) <= b <= a
        if turns > 64:
            assert b == a
        if turns < 0.5:
            assert b == pytest.approx(a / 40)
    assert all(x >= z for x, z in zip(y, y[1:]))


def test_turns_reduce_exactly():
    """position * turns modulo 2^64 against the same product in whole numbers of any size."""
    from fractions import Fraction
    freq = T.rotary_frequencies(128)[0]
    for f, t in zip(freq, T.turns_of(freq)):
        u = t % 2**64
        for pos in (0, 1, 4095, 2**31 - 1, 2**40 + 12345, -3):
            exact = pos * Fraction(f / (2 * math.pi)) % 1
            got = Fraction(pos * u % 2**64, 2**64)
            off = min(abs(exact - got), 1 - abs(exact - got))
            assert off <= Fraction(abs(pos) + 1, 2**64)


@pytest.mark.parametrize("bad", [dict(dim=3), dict(dim=0), dict(dim=64, base=1.0), dict(dim=64, scaling="other"),
                                 dict(dim=64, scaling="linear", factor=0.5), dict(dim=2, scaling="ntk", factor=2.0),
                                 dict(dim=64, scaling="yarn", beta_slow=0.0), dict(dim=64, base=math.nan)])
def test_frequency_refusals(bad):
    dim = bad.pop("dim")
    with pytest.raises(ValueError):
        T.rotary_frequencies(dim, **bad)


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the behaviour on a machine without CUDA")
def test_no_cpu_fallback():
    for f in (lambda: T.Rotary(64), lambda: T.PagedKVCache(4, 2, 64), lambda: T.Rotary(64, device="cpu")):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            f()
    i32 = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        T.PagedBatch(i32, i32[:1], i32[None, :1], 1)


def test_tensors_that_forward_mode_follows_are_refused():
    """Dual tensors, with gradients off too; plain ones within a level are not."""
    from torch.autograd import forward_ad
    x = torch.ones(3)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones(3))
        T._no_grad(x, x)
        with pytest.raises(ValueError, match="forward-mode"):
            T._no_grad(x, dual)
        with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
            T._no_grad(dual * 2)
    T._no_grad(x)


def _cache(**kw):
    a = 1 << 20
    d = dict(pages=8, kv_heads=2, key_dim=128, value_dim=128, k=a, v=a, k_scale=a, v_scale=a, status=a)
    d.update(kw)
    return _lib.EvaKvCache(*d.values())


def _batch(**kw):
    a = 1 << 20
    d = dict(seqs=3, tokens=3, max_q=1, max_pages=4, table_stride=4, q_start=a, seq_lens=a, table=a)
    d.update(kw)
    return _lib.EvaKvBatch(*d.values())


def test_entry_points_check_their_arguments_before_any_device_work():
    L, a, r = _lib.load(), 1 << 20, ctypes.byref
    rot = _lib.EvaRotary(64, 0, 0, 0, 1.0, 0, a)
    bad, ok = _lib.EVA_ERR_INVALID, _lib.EVA_OK

    def rotary(rot=rot, x=a, dtype=1, tokens=4, heads=2, dim=64, st=(128, 64), pos=a, out=a + 4096, so=(128, 64)):
        return L.eva_rotary(r(rot), x, dtype, tokens, heads, dim, *st, pos, 1, out, *so, None)

    assert rotary(tokens=0) == ok
    for kw in (dict(tokens=-1), dict(heads=0), dict(dim=62), dict(dtype=3), dict(x=None), dict(out=None), dict(pos=None),
               dict(x=a + 1), dict(pos=a + 4), dict(out=a, so=(64, 64)), dict(rot=_lib.EvaRotary(63, 0, 0, 0, 1.0, 0, a)),
               dict(rot=_lib.EvaRotary(32, 33, 0, 0, 1.0, 0, a)), dict(rot=_lib.EvaRotary(32, 34, 0, 0, 1.0, 0, a)),
               dict(rot=_lib.EvaRotary(32, 0, 0, 0, 1.0, 0, None)), dict(rot=_lib.EvaRotary(32, 0, 1, 0, 1.0, 0, a), st=(127, 64))):
        assert rotary(**kw) == bad, kw

    def append(c=None, b=None, rot=None, k=a, v=a, dtype=1):
        return L.eva_kv_append(r(c or _cache()), r(b or _batch()), None if rot is None else r(rot), k, 256, 128, v, 256, 128, dtype, None)

    for kw in (dict(b=_batch(seqs=0)), dict(b=_batch(tokens=0)), dict(b=_batch(max_q=0))):
        assert append(**kw) == ok
    for kw in (dict(c=_cache(pages=0)), dict(c=_cache(key_dim=96)), dict(c=_cache(value_dim=64)), dict(c=_cache(k=None)),
               dict(c=_cache(k=a + 8)), dict(c=_cache(status=None)), dict(c=_cache(kv_heads=0)), dict(b=_batch(seqs=-1)),
               dict(b=_batch(max_pages=0)), dict(b=_batch(table=None)), dict(b=_batch(q_start=a + 2)), dict(dtype=2), dict(k=None),
               dict(v=a + 1), dict(rot=_lib.EvaRotary(64, 0, 0, 1, 1.0, 0, a)), dict(rot=_lib.EvaRotary(64, 66, 0, 0, 1.0, 0, a))):
        assert append(**kw) == bad, kw

    def attend(c=None, b=None, q=a, dtype=1, heads=4, st=(512, 128), scale=0.1, window=0, ws=a, n=1 << 40, out=a):
        return L.eva_kv_attend(r(c or _cache()), r(b or _batch()), q, dtype, heads, *st, scale, window, ws, n, out, None)

    for kw in (dict(b=_batch(seqs=0)), dict(b=_batch(tokens=0)), dict(b=_batch(max_q=0))):
        assert attend(**kw) == ok
    for kw in (dict(heads=3), dict(heads=0), dict(dtype=2), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf),
               dict(window=-1), dict(q=None), dict(out=None), dict(ws=None), dict(q=a + 8), dict(out=a + 8), dict(st=(513, 128)),
               dict(st=(512, 132)), dict(c=_cache(v_scale=a + 2))):
        assert attend(**kw) == bad, kw
    need = L.eva_kv_attend_workspace(r(_cache()), r(_batch()), 4)
    assert need > 0 and attend(n=need - 1) == _lib.EVA_ERR_WORKSPACE
    assert L.eva_kv_attend_workspace(r(_cache()), r(_batch()), 3) == 0


@pytest.mark.parametrize("dk", [64, 128, 192])
def test_append_moves_each_dimension_once_at_aligned_places(dk):
    """The key kernel's units of two pairs (restated): every dimension in one unit, and where it moves two or four neighbours at
    a time (pairs side by side, or halves of an even number of pairs) their first one is a multiple of as many."""
    def pair(inter, dim, off, i):
        if inter or dim == 0:
            return 2 * i, 2 * i + 1
        if i < dim // 2:
            return off + i, off + i + dim // 2
        d = 2 * (i - dim // 2)
        e = d if d < off else d + dim
        return e, e + 1

    for inter in (False, True):
        for dim in range(0, dk + 1, 2):
            for off in range(0, dk - dim + 1, 2):
                seen = []
                for u in range(dk // 4):
                    (a0, b0), (a1, b1) = pair(inter, dim, off, 2 * u), pair(inter, dim, off, 2 * u + 1)
                    seen += [a0, b0, a1, b1]
                    if inter or dim == 0:
                        assert a0 % 4 == 0 and (b0, a1, b1) == (a0 + 1, a0 + 2, a0 + 3)
                    elif dim % 4 == 0 and 2 * u < dim // 2:
                        assert a0 % 2 == 0 and b0 % 2 == 0 and (a1, b1) == (a0 + 1, b0 + 1)
                    elif dim % 4 == 0:
                        assert a0 % 2 == 0 and a1 % 2 == 0 and (b0, b1) == (a0 + 1, a1 + 1)
                assert sorted(seen) == list(range(dk))


def test_oracle_scale_exponent():
    for amax, e in ((448.0, 0), (448.0001, 1), (1.75, -8), (1.0, -8), (0.0, -126), (3.0e38, 120), (1e-40, -126)):
        assert A.scale_exponent(amax) == e, amax
        assert e == -126 or (amax <= 448 * 2.0**e and amax > 448 * 2.0 ** (e - 1))


def test_oracle_rotation_is_a_rotation():
    x = torch.randn(4, 2, 16, dtype=torch.float64)
    pos = torch.tensor([0, 1, 50, 9])
    f = T.rotary_frequencies(8)[0]
    for layout in ("half", "interleaved"):
        y = A.rotate(x, pos, f, 1.0, layout, 4)
        assert torch.allclose(A.rotate(y, pos, f, 1.0, layout, 4, inverse=True), x, atol=1e-12)
        assert torch.equal(y[..., :4], x[..., :4]) and torch.equal(y[..., 12:], x[..., 12:]) and torch.equal(y[0], x[0])
    # a quarter turn takes (1, 0) to (0, 1)
    e = torch.zeros(1, 1, 2, dtype=torch.float64)
    e[..., 0] = 1
    assert torch.allclose(A.rotate(e, torch.tensor([1]), [math.pi / 2]), torch.tensor([[[0.0, 1.0]]], dtype=torch.float64), atol=1e-15)
