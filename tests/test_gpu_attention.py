"""Attention operators on a B200 against their 64-bit forms: rotary positions, the append into the paged 8-bit cache,
attention over it, and the three together. Needs a GPU."""
import math

import pytest
import torch

from eva_b200 import _lib
from eva_b200.attention import PagedBatch, PagedKVCache, Rotary
from oracle import attention as A

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


# ---- rotary ---------------------------------------------------------------------------------------------------

def _check_rotation(x, pos, rot, got, inverse=False):
    """Angle: 2^-25 half turns (conversion of the fraction) is 1e-7; cosine and sine 1e-7 more, products and sum 1.2e-7 of
    |a| + |b|; then the output's own rounding, half a step of its type. Far out the 64-bit angle itself is rounded: the
    oracle's product by 2^-53 of it, the kernel's fraction of a turn by the division by 2 pi and that constant, 2^-53 each."""
    ref = A.rotate(x.cpu(), pos.cpu(), rot.inv_freq, rot.mscale, rot.layout, rot.offset, inverse)
    size = x.cpu().double().abs()
    lo, hi = rot.offset, rot.offset + rot.dim
    pair = size[..., lo:hi]
    if rot.layout == "half":
        both = (pair[..., :rot.dim // 2] + pair[..., rot.dim // 2:]).repeat(1, 1, 2)
    else:
        both = (pair[..., 0::2] + pair[..., 1::2]).repeat_interleave(2, -1)
    tol = torch.zeros_like(ref)
    far = float(pos.abs().max()) * max(rot.inv_freq) * 3 * 2.0**-53
    tol[..., lo:hi] = (3.5e-7 + far) * abs(rot.mscale) * both + torch.finfo(x.dtype).eps / 2 * ref[..., lo:hi].abs() \
        + torch.finfo(x.dtype).smallest_normal
    err = (got.cpu().double() - ref).abs()
    worst = float((err - tol).max())
    assert worst <= 0, worst


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("tokens,heads,dim,rot,offset", [(1, 1, 64, 64, 0), (3, 5, 80, 40, 8), (70, 16, 192, 64, 128),
                                                         (257, 3, 102, 6, 34), (9, 33, 128, 128, 0)])
def test_rotary_matches_64_bits(layout, dtype, tokens, heads, dim, rot, offset):
    g = torch.Generator(device=DEV).manual_seed(tokens)
    x = torch.randn(tokens, heads, dim, device=DEV, generator=g).to(dtype)
    pos = torch.randint(0, 1 << 21, (tokens,), device=DEV, generator=g)
    r = Rotary(rot, layout=layout, offset=offset)
    out = r.apply(x, pos)
    _check_rotation(x, pos, r, out)
    assert torch.equal(r.apply(x, pos.to(torch.int32)), out)
    y = x.clone()
    assert r.apply(y, pos, out=y) is y and torch.equal(y, out)
    _check_rotation(x, pos, r, r.apply(x, pos, inverse=True), inverse=True)


@pytest.mark.parametrize("scaling,kw", [("linear", dict(factor=8.0)), ("ntk", dict(factor=4.0)),
                                        ("yarn", dict(factor=40.0)), ("yarn", dict(factor=40.0, mscale=1.0))])
def test_rotary_scalings_at_far_positions(scaling, kw):
    r = Rotary(64, layout="interleaved", offset=64, scaling=scaling, **kw)
    x = torch.randn(40, 4, 128, device=DEV)
    pos = torch.randint(2**31 - 1000, 2**33, (40,), device=DEV)
    pos[0] = -5
    _check_rotation(x, pos, r, r.apply(x, pos))


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_strides_and_unaligned_rows(layout):
    """Slices of a wider projection, heads and tokens exchanged, a last dimension that is not contiguous, odd offsets."""
    r = Rotary(32, layout=layout, offset=2)
    pos = torch.arange(7, 18, device=DEV)
    wide = torch.randn(11, 500, device=DEV).to(BF16)
    for x in (wide[:, 3:3 + 6 * 48].unflatten(1, (6, 48)), wide[:, :6 * 48].unflatten(1, (6, 48)),
              wide[:, :288].unflatten(1, (6, 48)).transpose(0, 1).contiguous().transpose(0, 1),
              wide[:, :288].unflatten(1, (48, 6)).transpose(1, 2), wide[:, None, 1:49], wide[:, None, :48].expand(11, 4, 48)):
        _check_rotation(x, pos, r, r.apply(x, pos))
    out = torch.zeros(11, 6, 64, device=DEV, dtype=BF16)
    x = wide[:, :288].unflatten(1, (6, 48))
    r.apply(x, pos, out=out[..., 8:56])
    _check_rotation(x, pos, r, out[..., 8:56])
    assert not out[..., :8].any() and not out[..., 56:].any()


def test_rotary_inverse_is_the_gradient():
    """<w, R x> is linear in x: its gradient R^T w is the inverse rotation; against differences, exact but for rounding."""
    r = Rotary(48, layout="half", offset=4, scaling="yarn", factor=4.0)
    x, w = (torch.randn(5, 3, 64, device=DEV) for _ in range(2))
    pos = torch.tensor([0, 1, 77, 4096, 300000], device=DEV)
    grad = r.apply(w, pos, inverse=True)
    for t, h, d in ((0, 0, 0), (1, 2, 4), (2, 1, 28), (4, 2, 51), (3, 0, 52), (4, 1, 63)):
        e = torch.zeros_like(x)
        e[t, h, d] = 1.0
        diff = float((w.double() * (r.apply(x + e, pos).double() - r.apply(x - e, pos).double())).sum() / 2)
        # x +- e and the rotation are rounded: 64 terms, each within 3.5e-7 * 2 * 5
        assert abs(diff - float(grad[t, h, d])) < 5e-5, (t, h, d)


def test_rotary_of_nothing():
    r = Rotary(32, layout="half")
    x = torch.empty(0, 4, 64, device=DEV)
    assert r.apply(x, torch.empty(0, dtype=torch.int64, device=DEV)).shape == (0, 4, 64)


# ---- paged cache ----------------------------------------------------------------------------------------------

class Setup:
    """A cache full of old bytes (NaN codes among them), a shuffled page table and a ragged batch."""

    def __init__(self, dims, kv_heads, new, lens, seed=0, spare=2, rows_behind=0):
        self.g = torch.Generator().manual_seed(seed)
        dk, dv = dims
        each = [-(-n // A.PAGE) for n in lens]
        pages = sum(each) + spare
        order = torch.randperm(pages, generator=self.g).tolist()
        self.table = []
        for n in each:
            self.table.append(order[:n])
            order = order[n:]
        self.unused = order
        width = max(each + [1])
        self.new, self.lens = list(new), list(lens)
        self.start = [0]
        for n in new:
            self.start.append(self.start[-1] + n)
        self.T = self.start[-1] + rows_behind
        byte = lambda *s: torch.randint(0, 256, s, generator=self.g, dtype=torch.uint8)   # noqa: E731
        self.host = {"k": byte(pages, kv_heads, 64, dk).view(A.E4M3), "v": byte(pages, kv_heads, dv, 64).view(A.E4M3),
                     "ks": torch.randint(-12, 2, (pages, kv_heads, 4), generator=self.g),
                     "vs": torch.randint(-12, 2, (pages, kv_heads, 4), generator=self.g)}
        t = torch.full((len(lens), width), -1, dtype=torch.int32)
        for b, p in enumerate(self.table):
            t[b, :len(p)] = torch.tensor(p, dtype=torch.int32)
        self.cache = PagedKVCache(pages, kv_heads, dk, dv, k=self.host["k"].to(DEV), v=self.host["v"].to(DEV),
                                  k_scale=self.bytes_of("ks"), v_scale=self.bytes_of("vs"))
        self.batch = PagedBatch(torch.tensor(self.start, dtype=torch.int32, device=DEV),
                                torch.tensor(lens, dtype=torch.int32, device=DEV), t.to(DEV), max([*new, 0]))

    def bytes_of(self, name):
        return (self.host[name] + 127).to(torch.uint8).to(DEV)

    def fill(self, scale=1.0):
        """Every token of the sequences gets a finite key and value (what an append before would have left)."""
        for name, sn in (("k", "ks"), ("v", "vs")):
            for b, n in enumerate(self.lens):
                for i, p in enumerate(self.table[b]):
                    m = min(64, n - 64 * i)
                    c = self.host[name][p] if name == "k" else self.host[name][p].transpose(1, 2)
                    vals = (torch.randn(c.shape[0], m, c.shape[2], generator=self.g) * 120).clamp(-448, 448)
                    c.view(torch.uint8)[:, :m] = vals.to(A.E4M3).view(torch.uint8)
                    self.host[sn][p] = torch.randint(-9, -5, self.host[sn][p].shape, generator=self.g)
            getattr(self.cache, name).view(torch.uint8).copy_(self.host[name].view(torch.uint8))
            getattr(self.cache, name + "_scale").view(torch.uint8).copy_((self.host[sn] + 127).to(torch.uint8))
        return self

    def rows(self, heads, dim, dtype, scale=1.0):
        return (torch.randn(self.T, heads, dim, generator=self.g) * scale).to(dtype)


DIMS = [(64, 64), (128, 128), (192, 128)]
# new tokens and lengths: one token, block and page borders, an empty sequence, a padding row, contexts that end inside blocks
BATCHES = [([1], [1]), ([1, 1, 1, 1], [16, 17, 64, 65]), ([5, 0, 1, 33], [5, 70, 0, 130]), ([130], [130]),
           ([64, 1, 15], [100, 49, 300]), ([3, 20], [2, 20])]


def _same_bytes(got, want, name):
    g, w = got.cpu().view(torch.uint8), want.view(torch.uint8)
    nan = ((g & 0x7f) == 0x7f) & ((w & 0x7f) == 0x7f)
    assert bool(((g == w) | nan).all()), (name, int(((g != w) & ~nan).sum()))


@pytest.mark.parametrize("dims", DIMS)
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("new,lens", BATCHES)
def test_append_without_rotation_is_exact(dims, dtype, new, lens):
    s = Setup(dims, 3, new, lens, seed=len(lens))
    k, v = s.rows(3, dims[0], dtype, 3.0), s.rows(3, dims[1], dtype, 0.02)
    s.cache.append(k.to(DEV), v.to(DEV), s.batch)
    A.append(s.host, k.double(), v.double(), s.start, s.lens, s.table)
    for name in ("k", "v"):
        _same_bytes(getattr(s.cache, name), s.host[name], name)
        assert torch.equal(getattr(s.cache, name + "_scale").view(torch.uint8), s.bytes_of(name + "s"))
    assert s.cache.status() == 0


@pytest.mark.parametrize("dims,layout,rot,offset", [((64, 64), "half", 64, 0), ((128, 128), "interleaved", 44, 84),
                                                    ((128, 128), "half", 128, 0), ((192, 128), "interleaved", 64, 128),
                                                    ((192, 128), "half", 30, 2)])
def test_append_rotates_by_the_position_in_the_sequence(dims, layout, rot, offset):
    """Angle error 1e-7 and the fast functions' 5e-7 before the rounding to e4m3 (half a step: 2^-4 of the value, or
    2^-10 of the scale below its normal range); the scale is the exact one unless the largest key lies within that of a power of two."""
    new, lens = [40, 1, 7], [40, 100, 200007]
    s = Setup(dims, 2, new, lens, seed=rot)
    r = Rotary(rot, layout=layout, offset=offset, scaling="yarn", factor=8.0)
    k, v = s.rows(2, dims[0], BF16, 2.0), s.rows(2, dims[1], BF16)
    pos = torch.cat([torch.arange(n - m, n) for m, n in zip(new, lens)])
    kr = A.rotate(k, pos, r.inv_freq, r.mscale, layout, offset)
    ek, ev = A.append(s.host, kr, v.double(), s.start, s.lens, s.table)
    s.cache.append(k.to(DEV), v.to(DEV), s.batch, rotary=r)
    _same_bytes(s.cache.v, s.host["v"], "v")
    codes, e = s.cache.k.cpu().float(), s.cache.k_scale.cpu().view(torch.uint8).int() - 127
    for (p, h, t), want in ek.items():
        two = 2.0 ** int(e[p, h, t // 16])
        tol = want.abs() * 2.0**-4 + two * 2.0**-10 + 1e-6 * r.mscale * k.abs().max().double()
        assert bool(((codes[p, h, t].double() * two - want).abs() <= tol).all())
        assert abs(int(e[p, h, t // 16]) - int(s.host["ks"][p, h, t // 16])) <= 1
    moved = (e != s.host["ks"].int()).float().mean()
    assert float(moved) < 0.01


def test_append_step_by_step_equals_one_append():
    """The scale of a block does not depend on how its tokens arrive; codes may differ only where a rescaled one is subnormal."""
    n = 150
    a, b = Setup((128, 128), 2, [n], [n], seed=5), Setup((128, 128), 2, [n], [n], seed=5)
    k, v = a.rows(2, 128, BF16), a.rows(2, 128, BF16)
    k *= torch.rand(n, 1, 1, generator=a.g).to(BF16) * 30
    a.cache.append(k.to(DEV), v.to(DEV), a.batch)
    at = 0
    for step in (1, 1, 13, 2, 40, 7, 1, 16, 16, 53):
        i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)   # noqa: E731
        batch = PagedBatch(i32(0, step), i32(at + step), b.batch.table, step)
        b.cache.append(k[at:at + step].to(DEV), v[at:at + step].to(DEV), batch)
        at += step
    assert at == n
    pages = torch.tensor(a.table[0], device=DEV)
    for name in ("k_scale", "v_scale"):
        assert torch.equal(getattr(a.cache, name).view(torch.uint8)[pages, :], getattr(b.cache, name).view(torch.uint8)[pages, :])
    for x, y, sc in zip(a.cache.values(pages), b.cache.values(pages), (a.cache.k_scale, a.cache.v_scale)):
        x, y = x.transpose(1, 2).flatten(0, 1)[:n], y.transpose(1, 2).flatten(0, 1)[:n]
        step = sc[pages].float().repeat_interleave(16, -1).transpose(1, 2).flatten(0, 1)[:n, :, None] * 2.0**-9
        assert bool(((x - y).abs() <= step).all())


@pytest.mark.parametrize("dims", DIMS)
@pytest.mark.parametrize("layout,rot,offset", [("half", 40, 8), ("half", 22, 2), ("interleaved", 64, 0), (None, 0, 0)])
@pytest.mark.parametrize("kv_heads", [3, 19])
def test_append_of_rows_anywhere_in_memory(dims, layout, rot, offset, kv_heads):
    """The same bytes whether rows lie on 16 bytes (bulk copies), on 8, or on 2; whole and part blocks, more heads than warps."""
    dk, dv = dims
    new, lens = [1, 50, 16, 37], [9, 50, 48, 70]
    rotary = Rotary(rot, layout=layout, offset=offset) if rot else None
    want = None
    for shift in (0, 4, 1):
        s = Setup(dims, kv_heads, new, lens, seed=kv_heads)
        wide = torch.zeros(s.T, kv_heads * (dk + dv) + 8, dtype=BF16, device=DEV)
        wide[:, shift:shift + kv_heads * (dk + dv)] = s.rows(kv_heads, dk + dv, BF16).to(DEV).flatten(1)
        both = wide[:, shift:shift + kv_heads * (dk + dv)].unflatten(1, (kv_heads, dk + dv))
        s.cache.append(both[..., :dk], both[..., dk:], s.batch, rotary=rotary)
        assert s.cache.status() == 0
        got = [getattr(s.cache, n).view(torch.uint8).clone() for n in ("k", "v", "k_scale", "v_scale")]
        if want is None:
            want = got
            if rotary is None:
                k, v = both[..., :dk].cpu().double(), both[..., dk:].cpu().double()
                A.append(s.host, k, v, s.start, s.lens, s.table)
                _same_bytes(s.cache.k, s.host["k"], "k")
                _same_bytes(s.cache.v, s.host["v"], "v")
        assert all(torch.equal(a, b) for a, b in zip(got, want)), shift


@pytest.mark.parametrize("seqs,new,max_q", [(200, 1, 1 << 28), (3, 21, 1 << 28), (150, 2, 5000)])
def test_append_of_far_fewer_rows_than_max_q(seqs, new, max_q):
    """max_q only bounds the rows of a sequence: any one appends the same bytes."""
    got = []
    for bound in (new, max_q):
        s = Setup((64, 64), 2, [new] * seqs, [new + 7 * i for i in range(seqs)], seed=1)
        k, v = s.rows(2, 64, BF16).to(DEV), s.rows(2, 64, BF16).to(DEV)
        s.cache.append(k, v, PagedBatch(s.batch.q_start, s.batch.seq_lens, s.batch.table, bound))
        assert s.cache.status() == 0
        got.append([getattr(s.cache, n).view(torch.uint8).clone() for n in ("k", "v", "k_scale", "v_scale")])
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("dims", DIMS)
@pytest.mark.parametrize("size", [0.02, 200.0])
def test_append_beside_sequences_without_new_rows(dims, size):
    """Sequences that bring no row of their own touch nothing: many of them share the part-full page that one appends to (a forked
    prefix), one has no page at all, and the bytes are those of the append alone; at the larger size its scales grow."""
    idle, n, new = 60, 37, 3
    s = Setup(dims, 3, [new], [n + new], seed=9).fill()
    k, v = s.rows(3, dims[0], BF16, size), s.rows(3, dims[1], BF16, size)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)   # noqa: E731
    page = s.table[0][0]
    start = [0] * (idle + 1) + [new] * (idle + 2)
    lens = [n] * idle + [n + new] + [n] * idle + [n]
    table = [[page]] * (2 * idle + 1) + [[-1]]
    s.cache.append(k.to(DEV), v.to(DEV), PagedBatch(i32(start), i32(lens), i32(table), 64))
    A.append(s.host, k.double(), v.double(), s.start, s.lens, s.table)
    for name in ("k", "v"):
        _same_bytes(getattr(s.cache, name), s.host[name], name)
        assert torch.equal(getattr(s.cache, name + "_scale").view(torch.uint8), s.bytes_of(name + "s"))
    assert s.cache.status() == 0


def test_append_of_values_that_are_not_finite():
    """Such a token gets a NaN key; its block's other tokens and scales are as if it were not there, and so are its finite values."""
    s = Setup((64, 64), 2, [40], [70], seed=2)
    k, v = s.rows(2, 64, BF16), s.rows(2, 64, BF16)
    k[3, 0, 5], k[9, 1, 63], v[20, 0, 1], v[21, 1, 0] = math.inf, math.nan, -math.inf, math.nan
    s.cache.append(k.to(DEV), v.to(DEV), s.batch)
    A.append(s.host, k.double(), v.double(), s.start, s.lens, s.table)
    for name in ("k", "v"):
        _same_bytes(getattr(s.cache, name), s.host[name], name)
        assert torch.equal(getattr(s.cache, name + "_scale").view(torch.uint8), s.bytes_of(name + "s"))
    nan = s.cache.k.float().isnan()
    assert bool(nan[s.table[0][0], 0, 30 + 3].all()) and bool(nan[s.table[0][0], 1, 30 + 9].all())


@pytest.mark.parametrize("dtype,big,mscale", [(BF16, 2.0**124, 64.0), (F16, 1000.0, 2.0**120)])
@pytest.mark.parametrize("layout,rot,offset", [("half", 64, 0), ("interleaved", 20, 44), ("half", 22, 2)])
@pytest.mark.parametrize("shift", [0, 1])
def test_append_of_keys_that_the_rotation_takes_out_of_range(dtype, big, mscale, layout, rot, offset, shift):
    """A finite key that is not finite once rotated and scaled (|y| of a pair (a, a) is |a| mscale at least in one of the two) is
    treated as one that was not finite before: the same bytes."""
    r, got = Rotary(rot, layout=layout, offset=offset, mscale=mscale), []
    for value in (big, math.nan):
        s = Setup((64, 64), 3, [40, 3], [70, 23], seed=2)
        k, v = s.rows(3, 64, dtype), s.rows(3, 64, dtype)
        k[3, 0], k[11, 2], k[41, 1], k[42, 1] = value, value, value, value
        wide = torch.zeros(s.T, 3, 64 + 8, dtype=dtype, device=DEV)
        wide[:, :, shift:shift + 64] = k.to(DEV)
        s.cache.append(wide[:, :, shift:shift + 64], v.to(DEV), s.batch, rotary=r)
        got.append([getattr(s.cache, n).view(torch.uint8).clone() for n in ("k", "v", "k_scale", "v_scale")])
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_append_extremes_of_the_range():
    """Zero blocks, the smallest and the largest values of the input types."""
    for dtype, big, tiny in ((BF16, 3.0e38, 1e-38), (F16, 65504.0, 6e-8)):
        s = Setup((64, 64), 1, [64], [64], seed=3)
        k, v = s.rows(1, 64, dtype), s.rows(1, 64, dtype)
        k[:16], k[16:32], k[32:48] = 0.0, big, tiny
        v[:16], v[16:32], v[32:48] = tiny, 0.0, -big
        s.cache.append(k.to(DEV), v.to(DEV), s.batch)
        A.append(s.host, k.double(), v.double(), s.start, s.lens, s.table)
        for name in ("k", "v"):
            _same_bytes(getattr(s.cache, name), s.host[name], name)


# ---- attention ------------------------------------------------------------------------------------------------

def _check_attention(s, q, out, scale, window=0, lost=0.0):
    """Scores: key_dim products accumulated in 32 bits with truncation, 2^-23 of the sum of their sizes each at most; a query in
    8-bit parts drops 2^-18 of its largest element; weights rounded to 16 bits (2^-11) and the output to its type."""
    ref, mean_abs, size, loud = A.attend(s.host, q.cpu(), s.start, s.lens, s.table, scale, window)
    delta = q.shape[2] * 2.0**-23 * size + 2.0**-18 * loud + 2.0**-20
    tol = torch.finfo(q.dtype).eps / 2 * ref.abs() + mean_abs * (2.0**-11 + 2 * delta) + torch.finfo(q.dtype).smallest_normal + lost
    got = out.cpu().double()
    n = s.start[-1]
    err = (got - ref)[:n].abs()
    nan = ref[:n].isnan()
    assert torch.equal(got[:n].isnan(), nan)
    assert bool((err <= tol[:n])[~nan].all()), float((err - tol[:n])[~nan].max())


HEADS = [(1, 1), (4, 2), (6, 2), (8, 1), (15, 3)]


@pytest.mark.parametrize("dims", DIMS)
@pytest.mark.parametrize("heads,kv_heads", HEADS)
@pytest.mark.parametrize("new,lens", BATCHES)
def test_attention_matches_64_bits(dims, heads, kv_heads, new, lens):
    s = Setup(dims, kv_heads, new, lens, seed=heads).fill()
    q = s.rows(heads, dims[0], BF16 if heads % 2 else F16, 2.0).to(DEV)
    _check_attention(s, q, s.cache.attend(q, s.batch), dims[0] ** -0.5)
    assert s.cache.status() == 0


@pytest.mark.parametrize("window", [1, 16, 50, 64, 129, 1000])
@pytest.mark.parametrize("new,lens", [([1, 1, 1], [10, 129, 700]), ([90, 3], [300, 40]), ([200], [200])])
def test_attention_within_a_window(window, new, lens):
    s = Setup((128, 128), 2, new, lens, seed=window).fill()
    q = s.rows(6, 128, BF16, 2.0).to(DEV)
    _check_attention(s, q, s.cache.attend(q, s.batch, window=window, scale=0.2), 0.2, window)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("new,lens", [([1, 1], [3000, 77]), ([7], [1025]), ([150, 40], [1500, 40])])
def test_attention_over_longer_caches(dtype, new, lens):
    s = Setup((128, 128), 2, new, lens, seed=11).fill()
    q = s.rows(8, 128, dtype, 3.0).to(DEV)
    _check_attention(s, q, s.cache.attend(q, s.batch), 128 ** -0.5)


@pytest.mark.parametrize("new,lens", [([1], [500]), ([100], [100])])
@pytest.mark.parametrize("size", [1e-30, 1e-3, 1e4, 1e30])
def test_attention_of_very_large_and_small_queries(size, new, lens):
    """Softmax over equal scores, and over scores so far apart that one token has all the weight."""
    s = Setup((64, 64), 1, new, lens, seed=4).fill()
    q = s.rows(2, 64, BF16, size).to(DEV)
    out = s.cache.attend(q, s.batch)
    if size <= 1e-3:
        _check_attention(s, q, out, 0.125)
    else:
        ref, _, _, _ = A.attend(s.host, q.cpu(), s.start, s.lens, s.table, 0.125)
        # the largest score wins unless two lie within the scores' own error: bound by the values' range
        assert bool(out.isfinite().all()) and float((out.cpu().double() - ref).abs().median()) < 2.0**-8


def _tokens(s, b, h):
    """Keys and values of sequence b and head h as the cache's codes and scales give them, float64 [length, dim]."""
    two = lambda e: torch.exp2(e.double()).repeat_interleave(A.BLOCK, -1)   # noqa: E731
    pages = torch.tensor(s.table[b])
    K = s.host["k"][pages, h].double() * two(s.host["ks"][pages, h])[..., None]
    V = s.host["v"][pages, h].double() * two(s.host["vs"][pages, h])[:, None, :]
    return K.flatten(0, 1)[:s.lens[b]], V.transpose(1, 2).flatten(0, 1)[:s.lens[b]]


@pytest.mark.parametrize("new,lens", [([1, 1], [500, 70]), ([100], [100]), ([70, 60], [800, 300])])
@pytest.mark.parametrize("size", [1e4, 1e30])
def test_rows_of_large_scores_are_the_value_of_the_largest(size, new, lens):
    """A score is off by key_dim * 2^-23 of the sum of its products' sizes at most, and by 2^-25 of the query's largest element times the
    sum of the key's (its rounding to 16 bits). A row whose largest score leads by twice that and 20 more has all its weight on one
    token, but for 2e-9 of each other one: its value to half a step of the output's type and 2^-11 (the weight's 16 bits)."""
    s = Setup((64, 64), 2, new, lens, seed=4).fill()
    q = s.rows(4, 64, BF16, size)
    out = s.cache.attend(q.to(DEV), s.batch).cpu().double()
    clear = 0
    for b, n in enumerate(lens):
        for h in range(4):
            K, V = _tokens(s, b, h // 2)
            for i in range(new[b]):
                pos, row = n - new[b] + i, s.start[b] + i
                Q = q[row, h].double()
                x = 0.125 * K[:pos + 1] @ Q
                off = 0.125 * (64 * 2.0**-23 * (K[:pos + 1].abs() @ Q.abs()).max()
                               + 2.0**-25 * Q.abs().max() * K[:pos + 1].abs().sum(1).max())
                top = x.topk(min(2, pos + 1)).values
                if pos and float(top[0] - top[1]) <= 2 * float(off) + 20:
                    continue
                clear += 1
                want = V[int(x.argmax())]
                tol = want.abs() * (2.0**-9 + 2.0**-11 + 2.0**-20) + (pos + 1) * 2.1e-9 * V.abs().max()
                assert bool(((out[row, h] - want).abs() <= tol).all()), (b, h, i)
    assert clear >= 0.9 * 4 * sum(new)


@pytest.mark.parametrize("dims", [(64, 64), (128, 128)])
@pytest.mark.parametrize("new,lens", [([1, 3], [200, 700]), ([100, 40], [400, 700])])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_small_differences_of_large_scores(dims, new, lens, dtype):
    """Scores near +-20000, 5000 and 1000 that differ by a few units: one dimension of the keys is 448 throughout, another a whole number,
    the queries 2^10, 2^8 or 2^6 times the one and once the other, so that a product's sum has at most 19 bits and is exact.
    What is rounded is the exponent t of a weight, below 2^15 times log2(e): half a step is 2^-10 (the largest is rounded
    as t is, and cancels), ln 2 of it of each weight, in numerator and sum; then the weight's 16 bits, the output's products
    in 32 bits, and the output."""
    s = Setup(dims, 1, new, lens, seed=12).fill()
    g = torch.Generator().manual_seed(5)
    s.host["k"].view(torch.uint8).zero_()
    codes = s.host["k"]
    small = (torch.randn(codes.shape[:3], generator=g) * 20).round().clamp(-60, 60)
    codes.view(torch.uint8)[..., 3] = 0x7e   # 448
    codes.view(torch.uint8)[..., dims[0] - 2] = small.to(A.E4M3).view(torch.uint8)
    s.host["ks"].fill_(-7)
    for name, b in (("k", codes.view(torch.uint8)), ("k_scale", s.bytes_of("ks"))):
        getattr(s.cache, name).view(torch.uint8).copy_(b)
    q = torch.zeros(s.T, 6, dims[0], dtype=dtype)
    q[..., dims[0] - 2] = 1.0
    for h, big in enumerate((2.0**10, -2.0**10, 2.0**8, -2.0**8, 2.0**6, -2.0**6)):
        q[:, h, 3] = big
    scale = 5.5   # 448 * 2^10 * 2^-7 * 5.5 = 19712
    out = s.cache.attend(q.to(DEV), s.batch, scale=scale).cpu().double()
    ref, mean_abs, _, _ = A.attend(s.host, q, s.start, s.lens, s.table, scale)
    tol = torch.finfo(dtype).eps / 2 * ref.abs() + torch.finfo(dtype).smallest_normal \
        + mean_abs * (2.0**-11 + 2 * math.log(2) * 2.0**-10 + max(lens) * 2.0**-23)
    assert bool(((out - ref).abs() <= tol).all()), float(((out - ref).abs() - tol).max())


@pytest.mark.parametrize("new,lens", [([1, 1], [200, 700]), ([100, 40], [400, 700])])
def test_scores_beyond_32_bits(new, lens):
    """Above the range a row is NaN; below it a score has no weight, and a row of none but such is zero; the rows beside are right."""
    s = Setup((64, 64), 1, new, lens, seed=3).fill()
    s.host["k"].view(torch.uint8).fill_(0x7e)   # 448
    s.host["ks"].fill_(100)
    for b, n in enumerate(lens):   # every third token's keys are zero, but in the last sequence
        for t in range(0, n if b == 0 else 0, 3):
            s.host["k"].view(torch.uint8)[s.table[b][t // 64], 0, t % 64] = 0
    s.cache.k.view(torch.uint8).copy_(s.host["k"].view(torch.uint8))
    s.cache.k_scale.view(torch.uint8).copy_(s.bytes_of("ks"))
    q = torch.zeros(s.T, 4, 64, dtype=BF16)
    q[:, 0], q[:, 1], q[:, 2] = -2.0**30, 2.0**30, 2.0**-120   # scores -+2^141 and, of the others, 2^-8 and 0
    out = s.cache.attend(q.to(DEV), s.batch)
    ref, mean_abs, _, _ = A.attend(s.host, q, s.start, s.lens, s.table, 0.125)
    for h in (0, 2, 3):
        want = ref[:, h].clone()
        if h == 0:
            want[s.start[1]:] = 0.0
        tol = 2.0**-9 * want.abs() + mean_abs[:, h] * (2.0**-11 + 2.0**-12)
        assert bool(((out[:, h].cpu().double() - want).abs() <= tol).all()), h
    first = [s.start[b] + i for b in range(2) for i in range(new[b])]
    assert bool(out[first, 1].isnan().all())


@pytest.mark.parametrize("dims", DIMS)
@pytest.mark.parametrize("heads,kv_heads", [(4, 2), (15, 3)])
@pytest.mark.parametrize("new,lens", [([1, 1, 1], [16, 65, 1500]), ([5, 0, 33], [5, 70, 130]), ([130, 2], [700, 2000])])
def test_attention_within_the_rounding_of_its_operands(dims, heads, kv_heads, new, lens):
    """As above, with what the query's rounding to 16 bits can take at most, 2^-25 of its largest element, and half a step of a weight of
    16 bits (2^-28 of the largest) for each token whose own step that is."""
    s = Setup(dims, kv_heads, new, lens, seed=heads).fill()
    q = s.rows(heads, dims[0], BF16 if heads % 2 else F16, 2.0)
    q[:, :, ::7] *= 2.0**-9   # elements whose 16 bits end before the type's
    scale = dims[0] ** -0.5
    out = s.cache.attend(q.to(DEV), s.batch).cpu().double()
    ref, mean_abs, size, loud = A.attend(s.host, q, s.start, s.lens, s.table, scale)
    delta = dims[0] * 2.0**-23 * size + 2.0**-25 * loud + 2.0**-20
    tol = torch.finfo(q.dtype).eps / 2 * ref.abs() + torch.finfo(q.dtype).smallest_normal \
        + mean_abs * (2.0**-11 + 2 * delta) + max(lens) * 2.0**-28 * 448 * 2.0**-6
    assert bool(((out - ref).abs() <= tol).all()), float(((out - ref).abs() - tol).max())


@pytest.mark.parametrize("new,lens", [([1, 1, 1], [64, 200, 1500]), ([100, 40], [100, 700])])
@pytest.mark.parametrize("kind", ["first", "all", "blocks", "all but one", "tiny", "large"])
def test_attention_over_values_of_zero_and_of_very_different_sizes(kind, new, lens):
    """Tokens whose values are zero count in the softmax's sum all the same, wherever they lie. Of a block whose values are all below
    448 * 2^-48 the weights may round to nothing: then a row is off by no more than that, 2^-39."""
    dims = (64, 64)
    s = Setup(dims, 1, new, lens, seed=len(kind)).fill()
    v, e = s.host["v"].view(torch.uint8), s.host["vs"]
    for table, n in zip(s.table, lens):
        for i, page in enumerate(table):
            for block in range(4):
                at = 64 * i + 16 * block
                if kind == "tiny":
                    e[page, :, block] = (-126, -100, -60, -49, -48, -47, -8, -7)[(at // 16) % 8]
                elif kind == "large":
                    e[page, :, block] = (35, -30, 35, -126)[(at // 16) % 4]
                elif (kind == "all" or (kind == "first" and at < 128) or (kind == "blocks" and at // 16 % 3 != 1)
                      or (kind == "all but one" and at // 16 != n // 32)):
                    v[page, :, :, 16 * block:16 * block + 16] = 0
                    e[page, :, block] = -126
    s.cache.v.view(torch.uint8).copy_(s.host["v"].view(torch.uint8))
    s.cache.v_scale.view(torch.uint8).copy_(s.bytes_of("vs"))
    for heads, size in ((2, 0.1), (24, 2.0)):
        q = s.rows(heads, 64, BF16, size).to(DEV)
        _check_attention(s, q, s.cache.attend(q, s.batch), 0.125, lost=2.0**-39)


@pytest.mark.parametrize("new,lens", [([1, 3], [70, 200]), ([100, 3], [100, 200]), ([5], [2])])
def test_attention_extremes_of_its_arguments(new, lens):
    """A scale of zero (the mean of what a row sees), the longest window, queries of zero."""
    s = Setup((64, 64), 2, new, lens, seed=1).fill()
    q = s.rows(8, 64, BF16, 2.0).to(DEV)
    _check_attention(s, q, s.cache.attend(q, s.batch, scale=0), 0.0)
    _check_attention(s, q, s.cache.attend(q, s.batch, window=2**31 - 1), 0.125)
    _check_attention(s, q, s.cache.attend(q, s.batch, window=2**30), 0.125)
    q[::2] = 0
    _check_attention(s, q, s.cache.attend(q, s.batch), 0.125)


@pytest.mark.parametrize("heads", [17, 24, 64, 300])
def test_attention_of_many_heads_of_one_key(heads):
    """Single tokens whose query heads share one key and value are many rows of one sequence."""
    s = Setup((192, 128), 1, [1, 1, 0, 1], [1, 300, 20, 65], seed=heads).fill()
    q = s.rows(heads, 192, BF16, 2.0).to(DEV)
    _check_attention(s, q, s.cache.attend(q, s.batch), 192 ** -0.5)


def test_attention_keeps_rows_behind_the_last_sequence():
    for new, lens in (([1, 1], [30, 40]), ([70, 20], [100, 20])):
        s = Setup((64, 64), 2, new, lens, rows_behind=5).fill()
        q = s.rows(4, 64, BF16).to(DEV)
        out = torch.full((s.T, 4, 64), 7.0, dtype=BF16, device=DEV)
        assert s.cache.attend(q, s.batch, out=out) is out
        assert bool((out[s.start[-1]:] == 7).all())
        _check_attention(s, q, out, 0.125)


@pytest.mark.parametrize("new,lens", [([1], [90]), ([90], [90])])
def test_a_nan_key_reaches_exactly_the_rows_that_see_it(new, lens):
    s = Setup((128, 128), 2, new, lens).fill()
    for t in (80, 89):
        s.host["k"].view(torch.uint8)[s.table[0][t // 64], 1, t % 64] = 0x7f
    s.cache.k.view(torch.uint8).copy_(s.host["k"].view(torch.uint8))
    q = s.rows(4, 128, BF16).to(DEV)
    out = s.cache.attend(q, s.batch)
    _check_attention(s, q, out, 128 ** -0.5)
    if new[0] > 1:
        assert not out[:80].isnan().any() and bool(out[80:, 2:].isnan().all()) and not out[:, :2].isnan().any()


@pytest.mark.parametrize("new,lens", [([1, 1], [90, 90]), ([90, 30], [90, 70])])
def test_queries_that_are_not_finite_stay_in_their_rows(new, lens):
    s = Setup((64, 64), 2, new, lens).fill()
    q = s.rows(4, 64, BF16)
    q[0, 1, 3], q[s.start[1], 2, 0] = math.nan, math.inf
    out = s.cache.attend(q.to(DEV), s.batch)
    assert bool(out[0, 1].isnan().all()) and bool(out[s.start[1], 2].isnan().all())
    assert int(out.isnan().sum()) == 2 * 64


def test_workspace_sizes_kept_for_many_prompt_lengths():
    """A cache that sees many lengths and head counts keeps few sizes, each what the library asks for."""
    import ctypes
    s = Setup((64, 64), 2, [1], [100]).fill()
    for heads in (2, 8, 34):
        q = s.rows(heads, 64, BF16).to(DEV)
        for max_q in [*range(1, 40), 300, 5000, 1 << 28]:
            batch = PagedBatch(s.batch.q_start, s.batch.seq_lens, s.batch.table, max_q)
            rows = min(max_q * heads // 2, 17)
            if max_q in (1, 2, 17, 1 << 28):
                _check_attention(s, q, s.cache.attend(q, batch), 0.125)
            else:
                s.cache.attend(q[:0], batch)
            want = s.cache.lib.eva_kv_attend_workspace(ctypes.byref(s.cache._c), ctypes.byref(batch._c), heads)
            assert s.cache._sizes[rows] == want
    assert len(s.cache._sizes) <= 18 and s.cache.status() == 0


def test_attention_strided_queries():
    s = Setup((128, 128), 2, [20, 1], [100, 30]).fill()
    wide = torch.randn(s.T, 900, device=DEV).to(BF16)
    for q in (wide[:, :512].unflatten(1, (4, 128)), wide[:, 4:516].unflatten(1, (4, 128)),
              wide[:, :512].unflatten(1, (128, 4)).transpose(1, 2), wide[:, None, :128].expand(s.T, 4, 128)):
        _check_attention(s, q, s.cache.attend(q, s.batch), 128 ** -0.5)


def test_repeated_calls_give_the_same_bits():
    for new, lens in (([1] * 9, [50, 3000, 7, 700, 64, 1, 129, 2000, 333]), ([300, 70], [2000, 70])):
        s = Setup((128, 128), 2, new, lens).fill()
        q = s.rows(8, 128, BF16).to(DEV)
        first = s.cache.attend(q, s.batch)
        for _ in range(3):
            assert torch.equal(first, s.cache.attend(q, s.batch))


@pytest.mark.parametrize("heads,seqs", [(2, 2500), (40, 300)])
def test_attention_of_many_sequences(heads, seqs):
    """More sequences than threads look through at once, some empty; two query heads (few rows) and forty (many)."""
    g = torch.Generator().manual_seed(seqs)
    lens = torch.randint(0, 40, (seqs,), generator=g).tolist()
    lens[seqs // 2] = 700
    new = [min(1, n) for n in lens]
    s = Setup((64, 64), 1, new, lens, seed=1).fill()
    q = s.rows(heads, 64, BF16, 2.0).to(DEV)
    _check_attention(s, q, s.cache.attend(q, s.batch), 0.125)
    assert s.cache.status() == 0


def test_attention_of_one_long_sequence_and_head():
    """One item in all the pieces of the GPU: their partial sums are joined in groups, and the groups."""
    for heads, new in ((1, 1), (24, 1), (2, 60)):
        n = 30000
        s = Setup((64, 64), 1, [new], [n], seed=heads).fill()
        q = s.rows(heads, 64, F16, 2.0).to(DEV)
        out = s.cache.attend(q, s.batch)
        _check_attention(s, q, out, 0.125)
        assert torch.equal(out, s.cache.attend(q, s.batch))


@pytest.mark.parametrize("new", [1, 3, 100])
def test_pages_beyond_32_bit_offsets(new):
    """The last pages of a cache of 4.6 GB of keys give what its first ones do, through a table that is a slice of a wider one."""
    pages, heads = 70000, 8
    assert pages * heads * 64 * 128 > 2**32
    cache = PagedKVCache(pages, heads, 128)
    g = torch.Generator().manual_seed(new)
    k, v = (torch.randn(130, heads, 128, generator=g).to(BF16).to(DEV) for _ in range(2))
    q = torch.randn(new, 2 * heads, 128, generator=g).to(BF16).to(DEV)
    int32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)   # noqa: E731
    rotary, outs = Rotary(128, layout="half"), []
    for ids in ([0, 2, 1], [pages - 1, pages - 3, pages - 2]):
        table = int32([[-1] + ids + [-1, -1]])[:, 1:4]
        cache.append(k, v, PagedBatch(int32([0, 130]), int32([130]), table, 130), rotary=rotary)
        outs.append(cache.attend(q, PagedBatch(int32([0, new]), int32([130]), table, new)))
    first, last = torch.tensor([0, 2, 1], device=DEV), torch.tensor([pages - 1, pages - 3, pages - 2], device=DEV)
    for t in (cache.k, cache.v, cache.k_scale, cache.v_scale):
        assert torch.equal(t.view(torch.uint8)[first], t.view(torch.uint8)[last])
    assert torch.equal(*outs) and bool(outs[0].float().abs().sum() > 0)
    assert not cache.k.view(torch.uint8)[3:pages - 3:997].any() and cache.status() == 0


def test_two_layers_in_one_graph_and_two_graphs_in_turn():
    """Graphs that share a memory pool, replayed in turn, each with the other's contents in between."""
    s = Setup((128, 128), 2, [1, 1, 1], [65, 300, 1], seed=3).fill()
    big = Setup((128, 128), 2, [40, 3], [140, 90], seed=4).fill()
    qs, qb = s.rows(8, 128, BF16, 2.0).to(DEV), big.rows(8, 128, BF16, 2.0).to(DEV)
    want = [s.cache.attend(qs, s.batch), big.cache.attend(qb, big.batch)]
    stream, pool, graphs, outs = torch.cuda.Stream(), torch.cuda.graph_pool_handle(), [], []
    stream.wait_stream(torch.cuda.current_stream())
    for setup, q in ((s, qs), (big, qb)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool, stream=stream):
            outs.append([setup.cache.attend(q, setup.batch) for _ in range(2)])
        graphs.append(graph)
    for _ in range(3):
        for graph, pair, w in zip(graphs, outs, want):
            for o in pair:
                o.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(o, w) for o in pair)


# ---- the three together, streams, graphs, refusals ------------------------------------------------------------

@pytest.mark.parametrize("dims,layout", [((128, 128), "half"), ((192, 128), "interleaved")])
def test_a_conversation_of_prompt_and_steps(dims, layout):
    """Append and attend a prompt, a second piece, then single tokens, as one cache would be used."""
    total, kvh, heads = 150, 2, 6
    s = Setup(dims, kvh, [total], [total], seed=8)
    rot = 64
    r = Rotary(rot, layout=layout, offset=dims[0] - rot)
    k, v, q = s.rows(kvh, dims[0], BF16), s.rows(kvh, dims[1], BF16), s.rows(heads, dims[0], BF16, 2.0)
    pos = torch.arange(total)
    qr = r.apply(q.to(DEV), pos.to(DEV))
    at = 0
    for n in (70, 37, 1, 1, 2, 1):
        i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)   # noqa: E731
        batch = PagedBatch(i32(0, n), i32(at + n), s.batch.table, n)
        s.cache.append(k[at:at + n].to(DEV), v[at:at + n].to(DEV), batch, rotary=r)
        out = s.cache.attend(qr[at:at + n], batch)
        # the oracle reads the codes that the cache holds: the append has its own tests
        for name, sn in (("k", "ks"), ("v", "vs")):
            s.host[name] = getattr(s.cache, name).cpu()
            s.host[sn] = getattr(s.cache, name + "_scale").cpu().view(torch.uint8).int() - 127
        s.start, s.lens = [0, n], [at + n]
        _check_attention(s, qr[at:at + n], out, dims[0] ** -0.5)
        at += n
    assert s.cache.status() == 0


def test_graph_replay_with_new_contents():
    """A captured step of padded batch size: rotate, append, attend; replayed as lengths grow, one slot empty."""
    lens = [63, 0, 130]
    a, b = Setup((64, 64), 2, [1, 1, 1], [l + 8 for l in lens], seed=6), Setup((64, 64), 2, [1, 1, 1], [l + 8 for l in lens], seed=6)
    a.fill(), b.fill()
    r = Rotary(64, layout="half")
    buf = [torch.zeros(3, h, 64, dtype=BF16, device=DEV) for h in (4, 2, 2)]
    pos = torch.zeros(3, dtype=torch.int64, device=DEV)

    def step(s):
        q = r.apply(buf[0], pos)
        s.cache.append(buf[1], buf[2], s.batch, rotary=r)
        return s.cache.attend(q, s.batch)

    zero = torch.zeros(3, dtype=torch.int32, device=DEV)
    a.batch.seq_lens.copy_(zero)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(a)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(a)
    for i in range(1, 5):
        now = torch.tensor([lens[0] + i, 0, lens[2] + i], dtype=torch.int32, device=DEV)
        for s in (a, b):
            s.batch.seq_lens.copy_(now)
        pos.copy_((now - 1).clamp(min=0))
        for t in buf:
            t.normal_()
        graph.replay()
        want = step(b)
        assert torch.equal(out, want) and not out[1].any()
        assert torch.equal(a.cache.k.view(torch.uint8), b.cache.k.view(torch.uint8))
        assert torch.equal(a.cache.v.view(torch.uint8), b.cache.v.view(torch.uint8))
    assert a.cache.status() == 0


def test_two_streams_at_once():
    """Two attentions over one cache on two streams: their workspaces are their own."""
    s = Setup((128, 128), 2, [1] * 6, [4000, 3000, 20, 700, 1, 2500]).fill()
    q1, q2 = (s.rows(8, 128, BF16).to(DEV) for _ in range(2))
    want = [s.cache.attend(q, s.batch) for q in (q1, q2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, q in enumerate((q1, q2)):
            with torch.cuda.stream(streams[i]):
                got[i].append(s.cache.attend(q, s.batch))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


@pytest.mark.parametrize("new,lens", [([1] * 40, [3000 + 50 * i for i in range(40)]), ([300, 70], [2000, 5000])])
def test_a_timeout_of_an_earlier_call_does_not_spoil_later_ones(new, lens):
    """The status word keeps a timeout until it is cleared; calls in between give what they give without it (more pages than any cache
    level near the SMs holds, so that waits take their time), and leave the bit alone."""
    s = Setup((128, 128), 8, new, lens, seed=2).fill()
    k, v, q = (t.to(DEV) for t in (s.rows(8, 128, BF16), s.rows(8, 128, BF16), s.rows(32, 128, BF16, 2.0)))
    names = ("k", "v", "k_scale", "v_scale")
    before = [getattr(s.cache, n).view(torch.uint8).clone() for n in names]
    seen = []
    for bits in (0, _lib.STATUS_TIMEOUT):
        for n, b in zip(names, before):
            getattr(s.cache, n).view(torch.uint8).copy_(b)
        s.cache._status.fill_(bits)
        s.cache.append(k, v, s.batch)
        seen.append([s.cache.attend(q, s.batch) for _ in range(3)] + [getattr(s.cache, n).view(torch.uint8).clone() for n in names])
        assert s.cache.status() == bits
    assert all(torch.equal(a, b) for a, b in zip(*seen))


@pytest.mark.parametrize("new,lens", [([1, 1], [100, 200]), ([70, 40], [100, 200])])
def test_a_batch_that_does_not_fit_is_flagged_and_left_out(new, lens):
    """Page ids outside the cache, lengths beyond the table and row starts beyond the rows are bounded before any access
    (the index arithmetic has host tests): a status bit, no fault, and the other sequences' results stand."""
    s = Setup((64, 64), 2, new, lens).fill()
    q = s.rows(4, 64, BF16).to(DEV)
    good = s.cache.attend(q, s.batch)
    before = s.cache.k.view(torch.uint8).clone()
    k = torch.zeros(s.T, 2, 64, dtype=BF16, device=DEV)
    for broken in ("page", "negative", "length", "rows", "order"):
        t, sl, qs = s.batch.table.clone(), s.batch.seq_lens.clone(), s.batch.q_start.clone()
        if broken == "page":
            t[1, :] = s.cache.pages
        elif broken == "negative":
            t[1, :] = -7
        elif broken == "length":
            sl[1] = t.shape[1] * 64 + 1
        elif broken == "rows":
            qs[2] = s.T + 1
        else:
            qs[2] = qs[1] - 1
        bad = PagedBatch(qs, sl, t, max(new))
        out = s.cache.attend(q, bad)
        assert s.cache.status() == _lib.STATUS_BAD_BATCH, broken
        assert torch.equal(out[:s.start[1]], good[:s.start[1]]), broken
        s.cache.clear_status()
        sl[0] = 0
        s.cache.append(k, k, PagedBatch(qs, sl, t, max(new)))
        assert s.cache.status() == _lib.STATUS_BAD_BATCH, broken
        assert torch.equal(before, s.cache.k.view(torch.uint8)), broken
        s.cache.clear_status()


def test_layer_stack_with_attention(oracle):
    """MoEStack with attention halves, a prompt and then single tokens of two sequences, against the 64-bit forms layer by layer.
    The oracle attends over the codes that the caches hold: a key or value that differs by a rounding may fall to the next
    code, a whole step of e4m3, and the first token of a sequence carries that to its output with weight 1, so that no
    bound of single elements holds without it (the append has its own tests). Each layer rounds to BF16 nine times (two norms, rows of the
    projection, query, attention, its projection, the MoE's input, inner and output); a rounding moves a vector by at most 2^-9 of
    its 2-norm, and two roundings of neighbours by 2^-8: 18 x 2^-8 over two layers."""
    import numpy as np
    from eva_b200 import config as C
    from eva_b200.attention import make_attention
    from eva_b200.experts import make_layer
    from eva_b200.runner import EvaMoE
    from eva_b200.stack import MoEStack, make_norms
    cfg = C.MoEConfig("small", hidden=512, inter=256, n_experts=16, topk=4, router="sigmoid", n_group=4, topk_group=2,
                      route_scale=2.5, norm_topk=True, shared_inter=384, bits=3, shared_bits=4)
    L, H, heads, kvh, dk, dv = 2, cfg.hidden, 4, 2, 128, 128
    hosts = [make_layer(cfg, "cpu", seed=50 + i) for i in range(L)]
    r = Rotary(64, layout="interleaved", offset=64)
    att = make_attention(L, H, heads, kvh, dk, dv, 6, rotary=r, seed=3)
    norms, anorms = make_norms(L, H, DEV, seed=4), make_norms(L, H, DEV, seed=5)[:L]
    stack = MoEStack([EvaMoE(h.to(DEV), max_rows=48) for h in hosts], norms, attention=att, attention_norms=anorms)
    table = [[4, 1], [0, 3]]
    g = torch.Generator().manual_seed(1)
    f32 = lambda t: oracle.bf16_to_f32(t.contiguous().view(torch.int16).cpu().numpy().view(np.uint16))   # noqa: E731
    b16 = lambda a: torch.from_numpy(np.asarray(a, np.float32)).to(BF16).double().numpy()   # noqa: E731
    lens = [0, 0]
    for new in ([30, 12], [1, 1], [1, 1]):
        lens = [a + b for a, b in zip(lens, new)]
        start = [0, new[0], sum(new)]
        pos = torch.cat([torch.arange(n - m, n) for m, n in zip(new, lens)])
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)   # noqa: E731
        x = torch.randn(start[-1], H, generator=g).to(BF16)
        out = stack.forward(x.to(DEV), batch=PagedBatch(i32(start), i32(lens), i32(table), max(new)), positions=pos.to(DEV))
        resid = f32(x).astype(np.float64)
        for i in range(L):
            h = b16(oracle.rmsnorm(resid.astype(np.float32), f32(anorms[i]), 1e-6))
            rows = torch.from_numpy(b16(h @ f32(att[i].wqkv).astype(np.float64).T))
            q = rows[:, :heads * dk]
            q = A.rotate(q.unflatten(1, (heads, dk)), pos, r.inv_freq, 1.0, "interleaved", 64).to(BF16).double()
            c = att[i].cache
            host = {"k": c.k.cpu(), "v": c.v.cpu(), "ks": c.k_scale.cpu().view(torch.uint8).int() - 127,
                    "vs": c.v_scale.cpu().view(torch.uint8).int() - 127}
            o, _, _, _ = A.attend(host, q, start, lens, table, dk ** -0.5)
            resid = resid + b16(b16(o.flatten(1).numpy()) @ f32(att[i].wo).astype(np.float64).T)
            h = oracle.f32_to_bf16(oracle.rmsnorm(resid.astype(np.float32), f32(norms[i]), 1e-6))
            resid = resid + oracle.layer_forward(h, hosts[i])[0]
        ref = oracle.rmsnorm(resid.astype(np.float32), f32(norms[-1]), 1e-6)
        got = f32(out)
        err = float(np.linalg.norm(got - ref) / np.linalg.norm(ref))
        assert err <= 18 * 2.0**-8, (new, err)
    assert all(a.cache.status() == 0 for a in att)
    with pytest.raises(ValueError):
        stack.forward(x.to(DEV))
    with pytest.raises(ValueError):
        MoEStack(stack.layers, norms, attention=att)


def _leave_in_memory(value, *shapes):
    """Freed blocks full of `value` where the next tensors of these shapes are likely to lie."""
    blocks = [torch.full(shape, value, dtype=BF16, device=DEV) for shape in shapes for _ in range(40)]
    torch.cuda.synchronize()
    del blocks


@pytest.mark.parametrize("new,lens", [([1, 1, 1], [30, 70, 5]), ([40, 3, 1], [60, 70, 5])])
def test_attention_half_gives_zeros_to_rows_of_no_sequence(new, lens):
    """Rows behind the last sequence, and those of a sequence that does not fit its batch, come out of the layer half as
    zeros whatever the memory held before; the other rows' bits do not depend on it."""
    from eva_b200.attention import make_attention
    heads, dv, T = 4, 128, sum(new) + 5
    half = make_attention(1, 256, heads, 2, 128, dv, 8, seed=1)[0]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)   # noqa: E731
    start = [0, new[0], new[0] + new[1], sum(new)]
    batch = PagedBatch(i32(start), i32(lens), i32([[0, 1], [2, 3], [77, 77]]), max(new))
    h = torch.randn(T, 256, generator=torch.Generator().manual_seed(2)).to(BF16).to(DEV)
    positions = torch.zeros(T, dtype=torch.int64, device=DEV)
    batch.seq_lens[2] = 129   # longer than its pages
    seen = []
    for value in (math.nan, 3.0, 0.0):
        _leave_in_memory(value, (T, heads, dv), (T, 256), (T, heads * 128 + 512))
        out32 = torch.empty(T, 256, device=DEV)
        seen.append((half.forward(h, batch, positions), half.forward(h, batch, positions, out_f32=out32).clone()))
        assert half.cache.status() == _lib.STATUS_BAD_BATCH
        half.cache.clear_status()
        for y in seen[-1]:
            assert bool(y.isfinite().all()) and not y[start[2]:].any() and bool(y[:start[2]].any(1).all())
    for other in seen[1:]:
        assert all(torch.equal(a, b) for a, b in zip(seen[0], other))


@pytest.mark.parametrize("new,lens", [([1, 1], [1, 1]), ([40, 3], [40, 3])])
def test_attention_half_keeps_32_bits_where_they_are_asked_for(new, lens):
    """out_f32 is the product of the attention's BF16 output and wo with nothing rounded but its 32-bit sums: 64 terms, each within
    2^-23 of the terms' sizes (a BF16 result is off by up to 2^-9 of the sum)."""
    from eva_b200.attention import make_attention
    half = make_attention(1, 96, 1, 1, 64, 64, 4, seed=1)[0]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)   # noqa: E731
    T = sum(new)
    batch, pos = PagedBatch(i32([0, new[0], T]), i32(lens), i32([[0], [1]]), max(new)), torch.zeros(T, dtype=torch.int64, device=DEV)
    h = torch.randn(T, 96, generator=torch.Generator().manual_seed(2)).to(BF16).to(DEV)
    wide = torch.empty(T, 200, device=DEV)
    out = half.forward(h, batch, pos, out_f32=wide[:, :96])
    assert out.data_ptr() == wide.data_ptr() and out.shape == (T, 96)
    o = half.cache.attend((h @ half.wqkv.T)[:, None, :64], batch).flatten(1).double()
    ref, size = o @ half.wo.T.double(), o.abs() @ half.wo.T.double().abs()
    assert bool(((out.double() - ref).abs() <= 64 * 2.0**-23 * size).all())
    y = half.forward(h, batch, pos)
    assert y.dtype == BF16 and bool(((y.double() - ref).abs() <= 64 * 2.0**-23 * size + 2.0**-8 * ref.abs() + 1e-38).all())
    half.wo.requires_grad_()
    half.forward(h, batch, pos, out_f32=torch.empty(T, 96, device=DEV)).sum().backward()
    want = o.sum(0)   # of the sum over the output: every row of wo has it, rounded to BF16
    assert bool(((half.wo.grad.double() - want).abs() <= 2.0**-7 * o.abs().sum(0)).all())
    for bad in (torch.empty(T, 95, device=DEV), torch.empty(T, 96, device=DEV, dtype=BF16), torch.empty(T, 96)):
        with pytest.raises(ValueError):
            half.forward(h, batch, pos, out_f32=bad)


def test_layer_stack_of_a_padded_step():
    """A step of three rows of which two belong to sequences, captured and replayed with the third left over: what memory held before
    reaches no row."""
    from eva_b200 import config as C
    from eva_b200.attention import make_attention
    from eva_b200.experts import make_layer
    from eva_b200.runner import EvaMoE
    from eva_b200.stack import MoEStack, make_norms
    cfg = C.MoEConfig("small", hidden=512, inter=256, n_experts=16, topk=4, router="sigmoid", n_group=4, topk_group=2,
                      route_scale=2.5, norm_topk=True, shared_inter=384, bits=3, shared_bits=4)
    att = make_attention(2, cfg.hidden, 4, 2, 128, 128, 6, seed=3)
    norms, anorms = make_norms(2, cfg.hidden, DEV, seed=4), make_norms(2, cfg.hidden, DEV, seed=5)[:2]
    stack = MoEStack([EvaMoE(make_layer(cfg, "cpu", seed=50 + i).to(DEV), max_rows=16) for i in range(2)], norms,
                     attention=att, attention_norms=anorms)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)   # noqa: E731
    batch, pos = PagedBatch(i32([0, 1, 2, 3]), i32([7, 9, 1]), i32([[4], [1], [2]]), 1), torch.zeros(3, dtype=torch.int64, device=DEV)
    x = torch.randn(3, cfg.hidden, generator=torch.Generator().manual_seed(1)).to(BF16).to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        stack.forward(x, batch=batch, positions=pos)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = stack.forward(x, batch=batch, positions=pos)
    outs = []
    for third in (math.nan, 1.0):
        batch.q_start.copy_(i32([0, 1, 2, 3]))
        x[2] = third
        graph.replay()   # the third row's sequence is there: its contents stay in the graph's memory
        batch.q_start.copy_(i32([0, 1, 2, 2]))
        x[2] = 0.5
        graph.replay()
        outs.append(out.clone())
    assert bool(outs[0].isfinite().all()) and torch.equal(*outs)


def test_outputs_that_autograd_follows_are_refused():
    """A result written into a tensor with a history would keep that history's gradient."""
    s = Setup((64, 64), 2, [1, 1], [10, 20]).fill()
    q, pos = s.rows(4, 64, BF16).to(DEV), torch.zeros(2, dtype=torch.int64, device=DEV)
    r, w = Rotary(64, layout="half"), torch.ones(2, 4, 64, dtype=BF16, device=DEV, requires_grad=True)
    for out in (w, w * 2):
        with pytest.raises(ValueError, match="no gradients"):
            r.apply(q, pos, out=out)
        with pytest.raises(ValueError, match="no gradients"):
            s.cache.attend(q, s.batch, out=out)
    with torch.no_grad():
        assert r.apply(q, pos, out=w) is w and s.cache.attend(q, s.batch, out=w) is w


def test_dual_tensors_are_refused():
    """No tangent is dropped in silence; the same calls with plain tensors go on within the level."""
    from torch.autograd import forward_ad
    s = Setup((64, 64), 2, [1, 1], [10, 20]).fill()
    q, k, pos = s.rows(4, 64, BF16).to(DEV), s.rows(2, 64, BF16).to(DEV), torch.zeros(2, dtype=torch.int64, device=DEV)
    r = Rotary(64, layout="half")
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))   # noqa: E731
        for f in (lambda: r.apply(dual(q), pos), lambda: s.cache.attend(dual(q), s.batch), lambda: s.cache.append(dual(k), k, s.batch),
                  lambda: s.cache.append(k, dual(k), s.batch)):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(ValueError, match="forward-mode"):
                    f()
        s.cache.append(k, k, s.batch)
        assert s.cache.attend(r.apply(q, pos), s.batch).shape == q.shape


def test_refusals():
    s = Setup((64, 64), 2, [1, 1], [10, 20]).fill()
    q, k = s.rows(4, 64, BF16).to(DEV), s.rows(2, 64, BF16).to(DEV)
    r = Rotary(64, layout="half")
    bad = [
        lambda: PagedKVCache(4, 2, 96), lambda: PagedKVCache(0, 2, 64), lambda: PagedKVCache(4, 2, 128, 64),
        lambda: PagedKVCache(4, 2, 64, k=torch.zeros(4, 2, 64, 64, device=DEV)),
        lambda: s.cache.attend(q.float(), s.batch), lambda: s.cache.attend(q[:, :3], s.batch),
        lambda: s.cache.attend(q[..., :32], s.batch), lambda: s.cache.attend(q.cpu(), s.batch),
        lambda: s.cache.attend(q, s.batch, window=-1), lambda: s.cache.attend(q, s.batch, window=1.5),
        lambda: s.cache.attend(q, s.batch, scale=math.nan), lambda: s.cache.attend(q, s.batch, scale=-1.0),
        lambda: s.cache.attend(q, None), lambda: s.cache.attend(q, s.batch, out=q),
        lambda: s.cache.attend(q, s.batch, out=torch.empty(2, 4, 64, device=DEV)),
        lambda: s.cache.append(k, k.half(), s.batch), lambda: s.cache.append(k[:1], k, s.batch),
        lambda: s.cache.append(q, q, s.batch), lambda: s.cache.append(k, k, s.batch, rotary=Rotary(128)),
        lambda: s.cache.append(k, k, s.batch, rotary=3),
        lambda: PagedBatch(s.batch.q_start, s.batch.seq_lens, s.batch.table[:1], 1),
        lambda: PagedBatch(s.batch.q_start.long(), s.batch.seq_lens, s.batch.table, 1),
        lambda: PagedBatch(s.batch.q_start.cpu(), s.batch.seq_lens, s.batch.table, 1),
        lambda: PagedBatch(s.batch.q_start, s.batch.seq_lens, s.batch.table, -1),
        lambda: r.apply(q, torch.zeros(2, device=DEV)), lambda: r.apply(q, torch.zeros(3, dtype=torch.int64, device=DEV)),
        lambda: r.apply(q[..., :32], torch.zeros(2, dtype=torch.int64, device=DEV)),
        lambda: r.apply(q, torch.zeros(2, dtype=torch.int64, device=DEV), out=q[:, :, :].transpose(0, 1)),
        lambda: r.apply(q.double(), torch.zeros(2, dtype=torch.int64, device=DEV)),
        lambda: r.apply(q, torch.zeros(2, dtype=torch.int64, device=DEV), out=q[:1].expand(2, 4, 64)),
        lambda: (lambda e: r.apply(e, torch.zeros(2, dtype=torch.int64, device=DEV), out=e))(q[:1].expand(2, 4, 64)),
        lambda: s.cache.attend(q, PagedBatch(s.batch.q_start, s.batch.seq_lens, s.batch.table, 0)),
        lambda: (lambda e: r.apply(e, torch.zeros(2, dtype=torch.int64, device=DEV), out=e))(q.view(-1).unfold(0, 256, 32)[:2].unflatten(1, (4, 64))),
        lambda: s.cache.attend(q, s.batch, scale=3e38),
        lambda: r.apply(q.detach().requires_grad_(), torch.zeros(2, dtype=torch.int64, device=DEV)),
        lambda: s.cache.attend(q.detach().requires_grad_(), s.batch),
        lambda: s.cache.append(k, k.detach().requires_grad_(), s.batch),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"case {i} was accepted")
