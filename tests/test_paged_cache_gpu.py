"""Rotary positions, cache append and paged decode attention on the GPU against
their formulas in 64 bits.

Tolerances, with u = 2^-24 (half a step of FP32, relative):

* Rotation.  The turn count is exact to about 2^-50; its fraction is rounded
  to FP32 (an angle error of at most pi u), and sine and cosine are within 2
  steps of 2^-23 of the FP32 range [-1, 1]: together under 8 u.  Two products
  and a sum round by u of their size each.  So |error| <= 10 u (|a| + |b|)
  before the result is rounded to its type, by half a step.
* Attention.  A score is a dot product of D products accumulated in FP32 and
  scaled: |error| <= (D + 4) u S with S = scale * sum |q_d K_d|, and the
  exponent's argument rounds by u |s| <= u S more, so a weight is off by the
  factor exp(2 (D + 6) u S_max) at most, about 2 (D + 6) u S_max for numerator
  and denominator together twice that; ex2.approx adds 2^-22 each.  The sums
  over n keys round by (n + 16) u each (numerator and denominator).  With
  A = sum p_j |V_j|: |error| <= A (4 (D + 6) u S_max + 2 (n + 16) u + 2^-20).
  A 16-bit kernel may hold the weights as a sum of two 16-bit values for the
  tensor cores: relative 2^-16 at most in BF16 and 2^-22 in FP16, and 2^-25
  absolute in FP16, where the smallest weights are subnormal; they add
  2^-16 A + 2^-25 sum |V_j| / sum w, with sum w >= 1.  Then the result is
  rounded to its type, by half a step (and half the smallest subnormal).
"""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

import operatorlib

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}


def names(t):
    return str(t).split(".")[-1]


def watchdog():
    code = ctypes.c_int()
    operatorlib.check("watchdog", operatorlib.capi().opl_read_and_clear_watchdog(code))
    return code.value


@pytest.fixture(autouse=True)
def clean_watchdog(cuda):
    watchdog()
    yield
    assert watchdog() == 0


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


# ------------------------------------------------------------------ formulas

def rotate64(x, positions, inv_freq, sections, adjacent, inverse=False):
    """The rotation in 64 bits, and (|a| + |b|) of each element's pair."""
    positions = positions.reshape(-1, x.shape[0])
    pairs = inv_freq.numel()
    axis = torch.cat([torch.full((n,), i) for i, n in enumerate(sections or [pairs])]).long()
    angle = (positions[axis.cuda()].double() * inv_freq.double()[:, None]).t()[:, None, :]
    cos, sin = angle.cos(), angle.sin() * (-1 if inverse else 1)
    i = torch.arange(pairs, device="cuda")
    first, second = (2 * i, 2 * i + 1) if adjacent else (i, i + pairs)
    a, b = x.double()[..., first], x.double()[..., second]
    out, size = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    out[..., first], out[..., second] = a * cos - b * sin, a * sin + b * cos
    size[..., first] = size[..., second] = a.abs() + b.abs()
    return out, size


def close(got, want, slack):
    eps = torch.finfo(got.dtype).eps / 2
    tol = slack + eps * (want.abs() + slack) + TINY[got.dtype]
    error = (got.double() - want).abs()
    assert bool((error <= tol).all()), (error - tol).max().item()


def rope_close(got, want, size):
    close(got, want, 10 * U * size)
    still = size == 0
    assert torch.equal(got.double()[still], want[still])  # copied, or zeros turned


def attention64(q, k_cache, v_cache, table, lens, scale):
    """Attention in 64 bits, and the slack of the docstring."""
    batch, heads, dim = q.shape
    kv_heads, page = k_cache.shape[2], k_cache.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    slack = torch.zeros_like(out)
    for b, n in enumerate(lens):
        if n <= 0:
            continue
        j = torch.arange(n, device="cuda")
        at = table[b].long()[j // page]
        keys = k_cache[at, j % page].double().repeat_interleave(heads // kv_heads, dim=1)
        values = v_cache[at, j % page].double().repeat_interleave(heads // kv_heads, dim=1)
        s = torch.einsum("hd,nhd->hn", q[b].double(), keys) * scale
        p = torch.softmax(s, dim=1)
        out[b] = torch.einsum("hn,nhd->hd", p, values)
        size = torch.einsum("hd,nhd->hn", q[b].double().abs(), keys.abs()).amax(1) * abs(scale)
        a = torch.einsum("hn,nhd->hd", p, values.abs())
        slack[b] = a * (4 * (dim + 6) * U * size[:, None] + 2 * (n + 16) * U + 2.0 ** -20)
        if q.dtype != torch.float32:
            slack[b] += 2.0 ** -16 * a + 2.0 ** -25 * values.abs().sum(0)
    return out, slack


class Paged:
    """A cache, a block table and lengths: pages in any order, unused table
    entries and unused tokens poisoned."""

    def __init__(self, lens, kv_heads, dim, page, dtype, seed, heads_first=False, spare=2,
                 poison=float("nan")):
        g = gen(seed)
        self.lens = lens
        used = [-(-n // page) for n in lens]
        total = sum(used) + spare
        shape = (total, kv_heads, page, dim) if heads_first else (total, page, kv_heads, dim)
        self.k, self.v = (randn(g, *shape, dtype=dtype) for _ in range(2))
        if heads_first:
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        order = torch.randperm(total, generator=g, device="cuda").int()
        width = max(1, max(used))
        self.table = torch.full((len(lens), width), -7, dtype=torch.int32, device="cuda")
        at = 0
        for b, n in enumerate(used):
            self.table[b, :n] = order[at:at + n]
            if lens[b] % page:
                last = order[at + n - 1].long()
                self.k[last, lens[b] % page:] = poison
                self.v[last, lens[b] % page:] = poison
            at += n
        self.k[order[at:].long()] = poison
        self.v[order[at:].long()] = poison
        self.seq_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")


def check_attention(ops, cache, heads, scale=None, seed=5, q=None):
    dim = cache.k.shape[3]
    q = randn(gen(seed), len(cache.lens), heads, dim, dtype=cache.k.dtype) if q is None else q
    got = ops.paged_attention(q, cache.k, cache.v, cache.table, cache.seq_lens, scale)
    assert got.shape == q.shape and got.dtype == q.dtype
    want, slack = attention64(q, cache.k, cache.v, cache.table, cache.lens,
                              dim ** -0.5 if scale is None else scale)
    close(got, want, slack)
    return got


# ---------------------------------------------------------------------- rope

@pytest.mark.parametrize("dtype", TYPES, ids=names)
@pytest.mark.parametrize("adjacent", [False, True], ids=["halves", "adjacent"])
@pytest.mark.parametrize("tokens,heads,dim,rot", [
    (1, 1, 2, 2), (1, 48, 128, 128), (3, 5, 64, 64), (2, 3, 71, 34), (7, 3, 80, 40), (5, 2, 96, 32),
    (4, 1, 256, 256), (9, 2, 192, 96), (2500, 12, 64, 64), (33, 3, 20, 12), (3, 2, 64, 0)])
def test_rope(ops, dtype, adjacent, tokens, heads, dim, rot):
    g = gen(tokens * dim + rot)
    x = randn(g, tokens, heads, dim, dtype=dtype)
    inv_freq = (10000.0 ** (-torch.arange(0, rot, 2, device="cuda") / max(rot, 1))).float()
    positions = torch.randint(0, 5000, (tokens,), generator=g, device="cuda")
    for inverse in (False, True):
        got = ops.rope(x, positions, inv_freq, [], adjacent, inverse)
        rope_close(got, *rotate64(x, positions, inv_freq, [], adjacent, inverse))


@pytest.mark.parametrize("dtype", TYPES, ids=names)
@pytest.mark.parametrize("sections", [[32], [16, 16], [16, 8, 8], [0, 20, 11, 1], [1, 31]])
def test_rope_axes(ops, dtype, sections):
    g = gen(sum(sections) + len(sections))
    x = randn(g, 37, 4, 64, dtype=dtype)
    inv_freq = (10000.0 ** (-torch.arange(0, 64, 2, device="cuda") / 64)).float()
    positions = torch.randint(-50, 3000, (len(sections), 37), generator=g, device="cuda")
    for adjacent in (False, True):
        got = ops.rope(x, positions, inv_freq, sections, adjacent)
        rope_close(got, *rotate64(x, positions, inv_freq, sections, adjacent))


def test_rope_far_positions(ops):
    """Angles of far and negative positions keep their fraction."""
    x = randn(gen(1), 6, 2, 64)
    inv_freq = (10000.0 ** (-torch.arange(0, 64, 2, device="cuda") / 64)).float()
    positions = torch.tensor([0, 1, 2 ** 20, 2 ** 31 + 12345, -(2 ** 20) - 1, 2 ** 24 + 1],
                             device="cuda")
    rope_close(ops.rope(x, positions, inv_freq), *rotate64(x, positions, inv_freq, [], False))


@pytest.mark.parametrize("dtype", TYPES, ids=names)
def test_rope_strides(ops, dtype):
    """Slices of a packed projection, transposed heads, an odd offset and an
    expanded head."""
    g = gen(3)
    inv_freq = (10000.0 ** (-torch.arange(0, 64, 2, device="cuda") / 64)).float()
    positions = torch.arange(19, device="cuda") + 100
    flat = randn(g, 19 * 9 * 64 + 1, dtype=dtype)
    views = [flat[:-1].view(19, 9, 64)[:, 4:7], flat[:-1].view(9, 19, 64).transpose(0, 1),
             flat[1:].view(19, 9, 64), flat[:19 * 64].view(19, 1, 64).expand(19, 3, 64),
             flat[:19 * 3 * 67].view(19, 3, 67)[..., 3:]]
    for x in views:
        rope_close(ops.rope(x, positions, inv_freq), *rotate64(x, positions, inv_freq, [], False))


@pytest.mark.parametrize("adjacent", [False, True], ids=["halves", "adjacent"])
def test_rope_gradient(ops, adjacent):
    """inverse is the gradient: against the formula (autograd of the rotation
    in 64 bits) and against central differences of the operator's own output
    along random directions."""
    g = gen(8)
    x, upstream = randn(g, 11, 3, 64), randn(g, 11, 3, 64)
    inv_freq = (10000.0 ** (-torch.arange(0, 48, 2, device="cuda") / 48)).float()
    positions = torch.randint(0, 3000, (2, 11), generator=g, device="cuda")
    sections = [10, 14]
    grad = ops.rope(upstream, positions, inv_freq, sections, adjacent, True)
    leaf = x.double().requires_grad_()
    rotate64(leaf, positions, inv_freq, sections, adjacent)[0].backward(upstream.double())
    size = rotate64(upstream, positions, inv_freq, sections, adjacent, True)[1]
    rope_close(grad, leaf.grad, size)
    for _ in range(4):
        step = randn(g, 11, 3, 64)
        up = ops.rope(x + step, positions, inv_freq, sections, adjacent).double()
        down = ops.rope(x - step, positions, inv_freq, sections, adjacent).double()
        difference = ((up - down) / 2 * upstream.double()).sum()
        # The rotation is linear: only roundings differ, of x +- step (u of
        # their size) and of each side's rotation (10 u of its pair, and u of
        # the result), summed over the elements without any cancellation.
        scale = 12 * U * (2 * (x.abs() + step.abs()).double().amax() * 2)
        assert abs(difference - (grad.double() * step.double()).sum()) <= \
            scale * upstream.double().abs().sum() + 12 * U * (step.double().abs() * 2 * size).sum()


def test_rope_in_place(cuda):
    """rope_into may write over its input, strided or not."""
    g = gen(4)
    packed = randn(g, 50, 9, 64, dtype=torch.bfloat16)
    before = packed.clone()
    inv_freq = (10000.0 ** (-torch.arange(0, 64, 2, device="cuda") / 64)).float()
    positions = torch.arange(50, device="cuda")
    x = packed[:, 2:5]
    want = rotate64(x, positions, inv_freq, [], False)
    operatorlib.rope_into(x, x, positions, inv_freq)
    rope_close(x, *want)
    assert torch.equal(packed[:, :2], before[:, :2]) and torch.equal(packed[:, 5:], before[:, 5:])


# ----------------------------------------------------------------- kv_append

@pytest.mark.parametrize("dtype", TYPES, ids=names)
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rot,page,packed,heads_first,adjacent", [
    (1, 1, 1, 2, 2, 1, False, False, False), (1, 32, 8, 128, 128, 16, True, False, False),
    (64, 8, 8, 64, 64, 16, True, True, False), (5, 6, 2, 80, 40, 24, False, True, True),
    (7, 3, 1, 71, 34, 3, True, False, False), (1500, 4, 2, 96, 96, 64, True, False, True),
    (3, 16, 1, 256, 128, 32, True, True, False), (4, 4, 2, 64, 0, 16, False, False, False)])
def test_kv_append(ops, dtype, tokens, heads, kv_heads, dim, rot, page, packed, heads_first,
                   adjacent):
    g = gen(tokens + dim)
    if packed:
        q, k, v = randn(g, tokens, heads + 2 * kv_heads, dim, dtype=dtype).split(
            [heads, kv_heads, kv_heads], dim=1)
    else:
        q, k, v = (randn(g, tokens, h, dim, dtype=dtype) for h in (heads, kv_heads, kv_heads))
    pages = -(-tokens // page) + 3
    shape = (pages, kv_heads, page, dim) if heads_first else (pages, page, kv_heads, dim)
    k_cache, v_cache = (randn(g, *shape, dtype=dtype) for _ in range(2))
    if heads_first:
        k_cache, v_cache = k_cache.transpose(1, 2), v_cache.transpose(1, 2)
    inv_freq = (10000.0 ** (-torch.arange(0, rot, 2, device="cuda") / max(rot, 1))).float()
    sections = [rot // 4, rot // 2 - rot // 4] if rot else []
    positions = torch.randint(0, 9000, (2, tokens) if rot else (tokens,), generator=g,
                              device="cuda")
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens].contiguous()
    slots[tokens // 2] = -1 if tokens > 1 else slots[0]  # padding, kept out of the cache
    kept = slots >= 0
    before_k, before_v = k_cache.clone(), v_cache.clone()
    got = ops.kv_append(q, k, v, k_cache, v_cache, slots, positions, inv_freq, sections, adjacent)
    rope_close(got, *rotate64(q, positions, inv_freq, sections, adjacent))
    where = (slots[kept] // page, slots[kept] % page)
    want, size = rotate64(k, positions, inv_freq, sections, adjacent)
    rope_close(k_cache[where], want[kept], size[kept])
    assert torch.equal(v_cache[where], v[kept])
    # Nothing else is touched.
    before_k[where], before_v[where] = k_cache[where], v_cache[where]
    assert torch.equal(k_cache, before_k) and torch.equal(v_cache, before_v)


def test_kv_append_bad_slot_is_reported(ops):
    """A slot past the cache is not followed; the others of the call are."""
    k_cache, v_cache = torch.zeros(2, 4, 1, 64, device="cuda"), torch.zeros(2, 4, 1, 64, device="cuda")
    q = randn(gen(2), 3, 2, 64)
    kv = randn(gen(3), 3, 1, 64)
    slots = torch.tensor([8, 7, 2 ** 62], device="cuda")
    ops.kv_append(q, kv, kv, k_cache, v_cache, slots, torch.zeros(3, dtype=torch.int64, device="cuda"),
                  torch.ones(32, device="cuda"))
    assert watchdog() == 0x6b01
    assert torch.equal(v_cache.view(8, 64)[7], kv[1, 0])
    assert not v_cache.view(8, 64)[:7].any() and not k_cache.view(8, 64)[:7].any()


def test_kv_append_refuses_one_cache_for_both(ops):
    cache = torch.zeros(2, 4, 1, 64, device="cuda")
    kv = randn(gen(3), 3, 1, 64)
    index = torch.arange(3, device="cuda")
    with pytest.raises(RuntimeError, match="must not share memory"):
        ops.kv_append(kv, kv, kv, cache, cache, index, index, torch.ones(32, device="cuda"))
    assert not cache.any()


# ----------------------------------------------------------- paged_attention

@pytest.mark.parametrize("dtype", TYPES, ids=names)
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (12, 12), (4, 2), (12, 4), (32, 8), (8, 1),
                                            (20, 2), (16, 1), (34, 2), (64, 1)])
def test_attention_head_layouts(ops, dtype, heads, kv_heads):
    check_attention(ops, Paged([33, 1, 0, 257], kv_heads, 64, 16, dtype, heads), heads)


@pytest.mark.parametrize("dtype", TYPES, ids=names)
@pytest.mark.parametrize("dim", [1, 2, 8, 20, 32, 40, 64, 71, 72, 80, 96, 128, 136, 160, 192, 200,
                                 255, 256])
def test_attention_head_dims(ops, dtype, dim):
    check_attention(ops, Paged([65, 300, 2], 2, dim, 16, dtype, dim), 4)


@pytest.mark.parametrize("dtype", TYPES, ids=names)
@pytest.mark.parametrize("page", [1, 3, 7, 8, 16, 24, 64, 100, 1000])
def test_attention_page_sizes(ops, dtype, page):
    """Pages that end inside a tile, and tiles that end inside a page."""
    check_attention(ops, Paged([1, 15, 16, 17, 130, 999], 2, 128, page, dtype, page,
                               heads_first=page % 2 == 0), 6)


@pytest.mark.parametrize("dtype", TYPES, ids=names)
@pytest.mark.parametrize("lens", [[1], [7], [8], [9], [4097], [20011], [1, 20000, 3], [0], [0, 0, 0],
                                  [0] * 20 + [5] + [0] * 20, list(range(300)), [1] * 700,
                                  [i % 7 * 3 for i in range(2100)]],
                         ids=lambda x: f"{len(x)}x{max(x)}")
def test_attention_lengths(ops, dtype, lens):
    """One token to long sequences, empty ones, ragged batches past one CTA's
    threads."""
    got = check_attention(ops, Paged(lens, 2, 64, 16, dtype, len(lens)), 8)
    for b, n in enumerate(lens):
        if n == 0:
            assert not got[b].any()


@pytest.mark.parametrize("dtype", TYPES, ids=names)
def test_attention_single_head_long(ops, dtype):
    """One unit cut over every CTA."""
    check_attention(ops, Paged([50001], 1, 128, 64, dtype, 1), 1)
    check_attention(ops, Paged([50001], 1, 128, 64, dtype, 2), 16)


@pytest.mark.parametrize("dtype", TYPES, ids=names)
@pytest.mark.parametrize("scale", [0.0, 1.0, -0.3, 4.0])
def test_attention_scale(ops, dtype, scale):
    """Flat, peaked and negated scores."""
    check_attention(ops, Paged([200, 3], 2, 64, 16, dtype, 9), 4, scale)


@pytest.mark.parametrize("dtype", TYPES, ids=names)
def test_attention_strides(ops, dtype):
    """q a slice of a packed projection; keys and values in one tensor; a cache
    on an odd offset; a table that is a slice."""
    g = gen(12)
    base = Paged([70, 31, 5], 2, 64, 16, dtype, 12)
    pages = base.k.shape[0]
    q = randn(g, 3, 8, 64, dtype=dtype)[:, 2:6]
    both = torch.stack([base.k, base.v], dim=1)
    base.k, base.v = both[:, 0], both[:, 1]
    check_attention(ops, base, 4, q=q)
    wide = torch.full((3, 40), -1, dtype=torch.int32, device="cuda")
    wide[:, 3:3 + base.table.shape[1]] = base.table
    base.table = wide[:, 3:3 + base.table.shape[1]]
    check_attention(ops, base, 4, q=q)
    odd = torch.empty(pages * 16 * 2 * 64 + 1, dtype=dtype, device="cuda")[1:]
    odd = odd.view(pages, 16, 2, 64).copy_(base.k)
    base.k = odd
    check_attention(ops, base, 4, q=q)
    padded = torch.zeros(pages, 16, 2, 67, dtype=dtype, device="cuda")[..., 2:66].copy_(base.v)
    base.v = padded
    check_attention(ops, base, 4, q=q)


@pytest.mark.parametrize("dtype", TYPES, ids=names)
def test_attention_shared_pages(ops, dtype):
    """Two sequences over the same pages (a shared prefix)."""
    cache = Paged([100, 100], 2, 64, 16, dtype, 13)
    cache.table[1, :4] = cache.table[0, :4]
    check_attention(ops, cache, 4)


@pytest.mark.parametrize("dtype", TYPES, ids=names)
def test_attention_unread_values_do_not_matter(ops, dtype):
    """What lies behind a sequence is not read: NaN, infinities and zeros there
    give the same bits."""
    got = []
    for poison in (0.0, float("nan"), float("inf")):
        cache = Paged([77, 1, 300], 2, 128, 16, dtype, 21, poison=poison)
        q = randn(gen(1), 3, 8, 128, dtype=dtype)
        got.append(ops.paged_attention(q, cache.k, cache.v, cache.table, cache.seq_lens))
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


@pytest.mark.parametrize("dtype", TYPES, ids=names)
def test_attention_infinities_and_nan_in_keys(ops, dtype):
    """As the formula has it: a key that scores -inf counts nothing, +inf or
    NaN makes the head NaN, and other heads and sequences keep their values."""
    cache = Paged([40, 40], 2, 64, 16, dtype, 22)
    q = randn(gen(1), 2, 4, 64, dtype=dtype)
    q[:, :, 0] = 1.0
    where = cache.table[0, 1].long()
    clean = ops.paged_attention(q, cache.k, cache.v, cache.table, cache.seq_lens)
    k = cache.k.clone()
    k[where, 3, 0, 0] = -math.inf  # sequence 0, key 19, key-value head 0
    got = ops.paged_attention(q, k, cache.v, cache.table, cache.seq_lens)
    without = cache.v.clone()
    keys = torch.arange(40, device="cuda")
    at = cache.table[0].long()[keys // 16]
    s = torch.einsum("hd,nd->hn", q[0, :2].double(), k[at, keys % 16, 0].double()) / 8
    want = torch.softmax(s, 1) @ without[at, keys % 16, 0].double()
    assert torch.isfinite(got).all()
    slack = attention64(q, cache.k, cache.v, cache.table, cache.lens, 0.125)[1]
    close(got[0, :2], want, slack[0, :2])
    assert torch.equal(got[0, 2:], clean[0, 2:]) and torch.equal(got[1], clean[1])
    for bad in (math.inf, math.nan):
        k[where, 3, 0, 0] = bad
        got = ops.paged_attention(q, k, cache.v, cache.table, cache.seq_lens)
        assert torch.isnan(got[0, :2]).all()
        assert torch.equal(got[0, 2:], clean[0, 2:]) and torch.equal(got[1], clean[1])


@pytest.mark.parametrize("dtype", TYPES, ids=names)
@pytest.mark.parametrize("heads", [2, 12, 32])
def test_attention_infinity_in_values(ops, dtype, heads):
    """An infinite value leaves its column not finite in the heads that read
    it, and nothing else changes."""
    cache = Paged([40, 40], 2, 64, 16, dtype, 25)
    q = randn(gen(1), 2, heads, 64, dtype=dtype)
    clean = ops.paged_attention(q, cache.k, cache.v, cache.table, cache.seq_lens)
    v = cache.v.clone()
    v[cache.table[1, 0].long(), 5, 1, 9] = math.inf
    got = ops.paged_attention(q, cache.k, v, cache.table, cache.seq_lens)
    assert not torch.isfinite(got[1, heads // 2:, 9]).any()
    same = torch.ones_like(got, dtype=torch.bool)
    same[1, heads // 2:, 9] = False
    assert torch.equal(got[same], clean[same])


@pytest.mark.parametrize("dtype", TYPES, ids=names)
def test_attention_bad_indices_are_reported(ops, dtype):
    """A page outside the cache is left out and reported; so is a length past
    the table's row, which is cut, and a negative one, which is empty."""
    cache = Paged([64, 30], 2, 64, 16, dtype, 23)
    q = randn(gen(1), 2, 4, 64, dtype=dtype)
    table = cache.table.clone()
    for bad in (-1, cache.k.shape[0], 2 ** 31 - 1, -2 ** 31):
        table[0, 3] = bad
        got = ops.paged_attention(q, cache.k, cache.v, table, cache.seq_lens)
        assert watchdog() == 0x6b02
        want, slack = attention64(q, cache.k, cache.v, cache.table, [48, 30], 0.125)
        close(got, want, slack)
    for bad, cut in ((65, 64), (2 ** 31 - 1, 64), (-1, 0), (-2 ** 31, 0)):
        lens = torch.tensor([bad, 30], dtype=torch.int32, device="cuda")
        got = ops.paged_attention(q, cache.k, cache.v, cache.table, lens)
        assert watchdog() == 0x6b03
        want, slack = attention64(q, cache.k, cache.v, cache.table, [cut, 30], 0.125)
        close(got, want, slack)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=names)
def test_attention_offsets_past_32_bits(ops, dtype):
    """Pages more than 2^32 bytes (and, in FP16, 2^32 elements) apart."""
    page, kv_heads, dim = 1024, 8, 128
    pages = 4200 if dtype == torch.float16 else 1100
    k = torch.zeros(pages, page, kv_heads, dim, dtype=dtype, device="cuda")
    cache = Paged([1500], kv_heads, dim, page, dtype, 24, spare=0)
    table = torch.tensor([[pages - 1, pages - 3]], dtype=torch.int32, device="cuda")
    k[table[0].long()] = cache.k[cache.table[0].long()]
    q = randn(gen(1), 1, 8, dim, dtype=dtype)
    got = ops.paged_attention(q, k, k, table, cache.seq_lens)
    want = ops.paged_attention(q, cache.k, cache.k, cache.table, cache.seq_lens)
    assert torch.equal(got, want)
    new = randn(gen(2), 1, 8, dim, dtype=dtype)
    slot = torch.tensor([(pages - 2) * page + 1000], device="cuda")
    zero = torch.zeros(1, dtype=torch.int64, device="cuda")
    v = torch.empty_like(k)
    ops.kv_append(new, new, new, k, v, slot, zero, torch.ones(0, device="cuda"))
    assert torch.equal(k[pages - 2, 1000], new[0]) and torch.equal(v[pages - 2, 1000], new[0])


# -------------------------------------------------- streams, graphs, repeats

def test_results_repeat_bit_for_bit(ops):
    cache = Paged([3000, 5, 9001, 0, 64], 4, 128, 16, torch.bfloat16, 31)
    q = randn(gen(1), 5, 16, 128, dtype=torch.bfloat16)
    first = ops.paged_attention(q, cache.k, cache.v, cache.table, cache.seq_lens)
    for _ in range(20):
        assert torch.equal(first, ops.paged_attention(q, cache.k, cache.v, cache.table,
                                                      cache.seq_lens))


@pytest.mark.parametrize("dtype", TYPES, ids=names)
def test_two_streams_at_once(ops, dtype):
    caches = [Paged([4000, 17, 1200], 2, 128, 16, dtype, 40 + i) for i in range(2)]
    qs = [randn(gen(50 + i), 3, 8, 128, dtype=dtype) for i in range(2)]
    want = [ops.paged_attention(q, c.k, c.v, c.table, c.seq_lens) for q, c in zip(qs, caches)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                c = caches[i]
                got[i].append(ops.paged_attention(qs[i], c.k, c.v, c.table, c.seq_lens))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert torch.equal(g, want[i])


def test_raw_helpers_on_another_stream(cuda):
    """The raw helpers with an explicit stream and workspace give the torch
    ops' results."""
    operatorlib.load_operatorlib()
    ops = torch.ops.operatorlib
    cache = Paged([500, 3], 2, 64, 16, torch.float16, 60)
    q = randn(gen(1), 2, 4, 64, dtype=torch.float16)
    inv_freq = (10000.0 ** (-torch.arange(0, 64, 2, device="cuda") / 64)).float()
    positions = torch.tensor([499, 2], device="cuda")
    slots = torch.stack([cache.table[0, 31] * 16 + 3, cache.table[1, 0] * 16 + 2]).long()
    kv = randn(gen(2), 2, 2, 64, dtype=torch.float16)
    k2, v2 = cache.k.clone(), cache.v.clone()
    rotated = ops.kv_append(q, kv, kv, cache.k, cache.v, slots, positions, inv_freq)
    want = ops.paged_attention(rotated, cache.k, cache.v, cache.table, cache.seq_lens)
    stream = torch.cuda.Stream()
    workspace = operatorlib.paged_attention_workspace(4, 2, 64, cuda)
    out, q_out = torch.empty_like(q), torch.empty_like(q)
    torch.cuda.synchronize()
    operatorlib.kv_append_into(q, kv, kv, q_out, k2, v2, slots, positions, inv_freq, stream=stream)
    operatorlib.paged_attention_into(q_out, k2, v2, cache.table, cache.seq_lens, out, workspace,
                                     stream=stream)
    stream.synchronize()
    assert torch.equal(q_out, rotated) and torch.equal(out, want)
    assert torch.equal(torch.nan_to_num(k2), torch.nan_to_num(cache.k))


@pytest.mark.parametrize("dtype", TYPES, ids=names)
@pytest.mark.parametrize("lens", [[9] * 2500, [700] * 90, [5000] * 3], ids=lambda x: f"{len(x)}x{x[0]}")
def test_next_launch_may_overwrite_the_inputs(ops, cuda, dtype, lens):
    """What follows on the stream may write over what the attention reads: no
    launch begins before it has ended, whether units are cut between CTAs (a
    second launch) or not (nothing for that launch to do)."""
    cache = Paged(lens, 4, 64, 16, dtype, 61)
    inv_freq = (10000.0 ** (-torch.arange(0, 64, 2, device="cuda") / 64)).float()
    zero = torch.zeros(len(lens), dtype=torch.int64, device="cuda")
    q = randn(gen(1), len(lens), 8, 64, dtype=dtype)
    other = randn(gen(2), len(lens), 8, 64, dtype=dtype)
    want = ops.paged_attention(q, cache.k, cache.v, cache.table, cache.seq_lens)
    workspace = operatorlib.paged_attention_workspace(8, 4, 64, cuda)
    outs = [torch.empty_like(q) for _ in range(6)]
    buffers = [q.clone() for _ in outs]
    torch.cuda.synchronize()
    for out, buffer in zip(outs, buffers):
        operatorlib.paged_attention_into(buffer, cache.k, cache.v, cache.table, cache.seq_lens,
                                         out, workspace)
        operatorlib.rope_into(other, buffer, zero, inv_freq)  # angle 0: a copy of `other`
    for out, buffer in zip(outs, buffers):
        assert torch.equal(out, want) and torch.equal(buffer, other)


class Decoder:
    """A decoding loop's buffers for one layer: the calls of one step as a
    serving program makes them, and the same step from the formulas."""

    def __init__(self, dtype, seed, batch=5, heads=8, kv_heads=2, dim=64, page=16, most=6):
        g = gen(seed)
        self.page, self.kv_heads, self.dim = page, kv_heads, dim
        self.table = torch.randperm(batch * most, generator=g, device="cuda").int().view(batch, most)
        shape = (batch * most, page, kv_heads, dim)
        self.k, self.v = (torch.full(shape, math.nan, dtype=dtype, device="cuda") for _ in "kv")
        self.inv_freq = (10000.0 ** (-torch.arange(0, dim, 2, device="cuda") / dim)).float()
        self.lens = torch.zeros(batch, dtype=torch.int32, device="cuda")
        self.packed = randn(g, batch, heads + 2 * kv_heads, dim, dtype=dtype)
        self.parts = [heads, kv_heads, kv_heads]
        self.slots = torch.zeros(batch, dtype=torch.int64, device="cuda")
        self.positions = torch.zeros(batch, dtype=torch.int64, device="cuda")

    def advance(self, rows):
        """One more token for the first `rows` sequences; the rest is padding."""
        active = torch.arange(len(self.lens), device="cuda") < rows
        self.positions.copy_(self.lens)
        column = (self.positions // self.page).clamp(max=self.table.shape[1] - 1)
        slots = self.table.gather(1, column[:, None])[:, 0].long() * self.page + \
            self.positions % self.page
        self.slots.copy_(torch.where(active, slots, torch.full_like(slots, -1)))
        self.lens += active.int()

    def step(self, ops):
        q, k, v = self.packed.split(self.parts, dim=1)
        q = ops.kv_append(q, k, v, self.k, self.v, self.slots, self.positions, self.inv_freq)
        return q, ops.paged_attention(q, self.k, self.v, self.table, self.lens)


@pytest.mark.parametrize("dtype", TYPES, ids=names)
def test_decoding_run(ops, dtype):
    """Prompt (rope and append of many tokens), then steps of a growing ragged
    batch with padding rows, against the formulas on the whole history."""
    d = Decoder(dtype, 70)
    g = gen(71)
    history = []
    for step in range(40):
        d.packed.copy_(randn(g, *d.packed.shape))
        d.advance(rows=5 if step < 20 else 3)
        q, out = d.step(ops)
        history.append((d.packed.clone(), d.positions.clone(), d.slots.clone()))
        rope_close(q, *rotate64(d.packed[:, :8], d.positions, d.inv_freq, [], False))
        want, slack = attention64(q, d.k, d.v, d.table, d.lens.tolist(), d.dim ** -0.5)
        close(out, want, slack)
    for packed, positions, slots in history:
        kept = slots >= 0
        where = (slots[kept] // d.page, slots[kept] % d.page)
        _, k, v = packed.split(d.parts, dim=1)
        want, size = rotate64(k, positions, d.inv_freq, [], False)
        rope_close(d.k[where], want[kept], size[kept])
        assert torch.equal(d.v[where], v[kept])


def test_decoding_step_in_a_graph(ops):
    """A captured step, replayed with new inputs, lengths and slots, gives the
    eager step's bits; two graphs with caches of their own run at once."""
    eager, captured = Decoder(torch.bfloat16, 80), [Decoder(torch.bfloat16, 80) for _ in range(2)]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    for d in captured:
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            d.slots.fill_(-1)
            d.step(ops)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(d.step(ops))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    g = gen(81)
    for step in range(20):
        x = randn(g, *eager.packed.shape)
        for d in (eager, *captured):
            d.packed.copy_(x)
            d.advance(rows=4)
        want = eager.step(ops)
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for q, out in outs:
            assert torch.equal(q, want[0]) and torch.equal(out, want[1])
