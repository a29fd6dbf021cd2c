"""GPU: paged attention and append where small differences count, against the
definitions in 64 bits; the helpers and their bounds are those of the tests of
the ordinary cases."""

import pytest
import torch

from preemptlm_b200 import PagedKVCache, _abi, ops

from .test_gpu_decoder_layer import make
from .test_gpu_paged_attention import BF, DEV, F8, attend64, check_attention, make_cache, make_table, rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("D,heads,group", [(64, 2, 8), (128, 2, 5), (128, 1, 16), (256, 2, 8), (256, 1, 16)])
def test_probabilities_keep_sixteen_bits(bits, D, heads, group):
    """Pairs of tokens with opposite values and nearly equal scores: the output is the small difference of their
    probabilities.  Bound: one rounding of the output (2^-8 of it), and 2^-15 of the sum of probability * |v|: sixteen
    bits of a probability (2^-17), and below 2e-5 for fp32 scores (|score| < 0.1), exponential and sums of up to 64
    tokens."""
    lengths, page = [2, 4, 16, 34, 64], 16
    table, total = make_table(lengths, page, 1)
    cache = make_cache(total, heads, page, D, bits, 2)
    cache.v[:, :, 1::2] = (-cache.v[:, :, 0::2].float()).to(cache.v.dtype)
    q = rand((len(lengths), heads * group, D), 5, 0.01)
    got = ops.paged_attention(cache, q, table, torch.tensor(lengths, dtype=torch.int32, device=DEV))
    ref, mag = attend64(cache, q, table, lengths)
    err = (got.double() - ref).abs()
    bound = ref.abs() * 2.0 ** -8 + mag * 2.0 ** -15
    assert bool((err <= bound).all()), float((err / bound).max())


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("D,heads,group", [(64, 2, 2), (128, 1, 16), (256, 2, 8)])
def test_rows_of_the_table(bits, D, heads, group):
    """Tokens that share table rows, in any order, equal the same call over a gathered table; a row outside the table is
    zero, and recorded unless its token is padding."""
    page, sequences = 16, 4
    table, total = make_table([300, 40, 0, 700], page, 1)
    cache = make_cache(total, heads, page, D, bits, 2)
    rows = torch.tensor([3, 0, 0, 1, 3, 2, 3, 0, 1], dtype=torch.int32, device=DEV)
    lengths = [700, 1, 300, 40, 33, 0, 16, 155, 17]
    n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    q = rand((len(lengths), heads * group, D), 5)
    ops.device_status()
    got = ops.paged_attention(cache, q, table, n, rows=rows)
    assert torch.equal(got, ops.paged_attention(cache, q, table[rows.long()], n))
    check_attention(got, *attend64(cache, q, table[rows.long()], lengths), bits)
    assert ops.device_status() == 0
    for outside in (-1, sequences, -(1 << 31), (1 << 31) - 1):
        at, none = torch.tensor([0, 5, 8], device=DEV), torch.tensor([-7, 0, -1], dtype=torch.int32, device=DEV)
        bad = rows.clone()
        bad[at] = outside
        padded = n.clone()
        padded[at] = none
        out = ops.paged_attention(cache, q, table, padded, rows=bad)
        assert ops.device_status() == 0  # padding tokens
        assert bool((out[at] == 0).all())
        keep = [1, 2, 3, 4, 6, 7]
        assert torch.equal(out[keep], got[keep])
        out = ops.paged_attention(cache, q, table, n, rows=bad)
        assert ops.device_status() == _abi.SG_ERR_CAPACITY
        assert bool((out[at] == 0).all()) and torch.equal(out[keep], got[keep])
    with pytest.raises(TypeError):
        ops.paged_attention(cache, q, table, n, rows=rows.long())
    with pytest.raises(TypeError):
        ops.paged_attention(cache, q, table, n, rows=rows[:3])


@pytest.mark.parametrize("padding_row", [-1, 2, 1 << 30])
def test_block_with_padding_tokens(padding_row):
    """A step padded to a fixed size, its padding tokens' rows outside the table: what the tokens alone give."""
    att = make(256, 4, 2, 64, 64, 16, 8, BF)
    table = torch.arange(8, device=DEV, dtype=torch.int32).view(2, 4)
    x, r = rand((7, 256), 1), rand((7, 256), 2, 2.0)
    rows = torch.tensor([0, 0, 1, 0, 1], dtype=torch.int32, device=DEV)
    pos = torch.tensor([0, 1, 0, 2, 1], dtype=torch.int32, device=DEV)
    live = torch.tensor([0, 1, 3, 4, 6], device=DEV)
    want, _ = att(x[live], r[live], table, pos, rows)
    all_rows = torch.full((7,), padding_row, dtype=torch.int32, device=DEV)
    all_pos = torch.full((7,), -1, dtype=torch.int32, device=DEV)
    all_rows[live], all_pos[live] = rows, pos
    ops.device_status()
    got, _ = att(x, r, table, all_pos, all_rows)
    assert ops.device_status() == 0
    assert torch.equal(got[live], want) and bool((got[[2, 5]] == 0).all())
    all_pos[2] = 3  # a token without a sequence: left out and reported, the others as they were
    got, _ = att(x, r, table, all_pos, all_rows)
    assert ops.device_status() == _abi.SG_ERR_CAPACITY
    assert torch.equal(got[live], want) and bool((got[[2, 5]] == 0).all())


def test_table_with_more_rows_than_tokens():
    """Append and attention take the same tables: a fixed one with a smaller step."""
    page = 16
    table, total = make_table([40, 40, 40, 40], page, 1)
    cache = make_cache(total, 2, page, 128, 16, 2)
    q, n = rand((2, 8, 128), 3), torch.tensor([33, 20], dtype=torch.int32, device=DEV)
    got = ops.paged_attention(cache, q, table, n)
    assert torch.equal(got, ops.paged_attention(cache, q, table[:2], n))
    check_attention(got, *attend64(cache, q, table[:2], [33, 20]), 16)
    with pytest.raises(TypeError):
        ops.paged_attention(cache, q, table[:1], n)
    att = make(256, 4, 2, 64, 64, 16, 8, BF)
    table = torch.arange(8, device=DEV, dtype=torch.int32).view(4, 2)
    x, r, pos = rand((2, 256), 1), rand((2, 256), 2, 2.0), torch.zeros(2, dtype=torch.int32, device=DEV)
    want, _ = att(x, r, table[:2], pos)
    got, _ = att(x, r, table, pos)
    assert torch.equal(got, want)


def test_positions_past_the_rotation_table():
    """A token whose position the append leaves out attends nothing, as a padding token does."""
    att = make(256, 4, 2, 64, 64, 16, 64, BF)
    att.cache.v.fill_(1.0)  # what a slot that was never written may hold
    table = torch.arange(64, device=DEV, dtype=torch.int32).view(2, 32)
    x, r = rand((2, 256), 1), rand((2, 256), 2, 2.0)
    last = att.rope.shape[0] - 1
    ops.device_status()
    for pos in (last + 1, last + 100, (1 << 31) - 1):
        at = torch.tensor([5, pos], dtype=torch.int32, device=DEV)
        got, _ = att(x, r, table, at)
        assert ops.device_status() == _abi.SG_ERR_SHAPE
        assert bool((got[1] == 0).all()) and bool(got[0].any())
    got, _ = att(x, r, table, torch.tensor([5, last], dtype=torch.int32, device=DEV))
    assert ops.device_status() == 0 and bool(got[1].any())


def test_rows_longer_than_the_limit():
    page = 16
    lengths = [40, 41, 39, 100, 0]
    table, total = make_table(lengths, page, 1)
    cache = make_cache(total, 2, page, 64, 16, 2)
    q, n = rand((5, 4, 64), 3), torch.tensor(lengths, dtype=torch.int32, device=DEV)
    ops.device_status()
    want = ops.paged_attention(cache, q, table, n)
    for most in (100, 1 << 40):
        assert torch.equal(ops.paged_attention(cache, q, table, n, max_length=most), want)
    assert ops.device_status() == 0
    got = ops.paged_attention(cache, q, table, n, max_length=40)
    assert ops.device_status() == _abi.SG_ERR_SHAPE
    assert torch.equal(got[[0, 2, 4]], want[[0, 2, 4]]) and bool((got[[1, 3]] == 0).all())
    with pytest.raises(ValueError):
        ops.paged_attention(cache, q, table, n, max_length=-1)


@pytest.mark.parametrize("shared", [True, False])
def test_wide_tables(shared):
    """Far more tokens in the table than in the rows: rows go by their lengths, around the cuts of the call too."""
    heads, page, D, width = 32, 16, 64, 8192 if shared else 20000
    B = 4500 if shared else 1900  # of 131072 (320000) tokens and 32 heads: 1.2e9 slices of 16
    n = torch.arange(B, device=DEV, dtype=torch.int32) * 37 % 41
    cache = make_cache(64, heads, page, D, 16, 2)
    table = torch.full((3 if shared else B, width), -1, dtype=torch.int32, device=DEV)
    table[:, :3] = torch.randint(64, (table.shape[0], 3), generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)
    rows = torch.arange(B, device=DEV, dtype=torch.int32) % 3 if shared else None
    q = rand((B, heads, D), 3)
    got = ops.paged_attention(cache, q, table, n, rows=rows)
    narrow = table[:, :3].contiguous()
    most = (1 << 30) // (heads * width)  # rows that are counted at a time
    assert most < B
    for first in (0, most - 25, B - 50):
        at = slice(first, first + 50)
        pages = narrow[at] if rows is None else narrow[rows[at].long()]
        check_attention(got[at], *attend64(cache, q[at], pages, n[at].tolist()), 16)


def test_longest_tables():
    """One row of the widest table that is taken."""
    cache = make_cache(8, 16, 1024, 64, 16, 2)
    table = torch.full((1, 1 << 20), -1, dtype=torch.int32, device=DEV)  # 2^30 tokens
    table[0, :4] = torch.tensor([3, 1, 7, 0])
    q, n = rand((1, 16, 64), 3), torch.tensor([4000], dtype=torch.int32, device=DEV)
    check_attention(ops.paged_attention(cache, q, table, n), *attend64(cache, q, table[:, :4], [4000]), 16)
    with pytest.raises(_abi.SlottedGLUError):
        ops.paged_attention(cache, q, torch.cat((table, table), dim=1), n)


@pytest.mark.parametrize("T", [0, 1, 2])
@pytest.mark.parametrize("width", [257, 260, 264])
def test_views_of_few_tokens(T, width):
    """Rows of a wider buffer, whatever its width: read in place, or copied, with one token as with two."""
    page, D = 16, 64
    views = [rand((3, width), 10 + i)[:, : h * D].view(3, h, D)[:T] for i, h in enumerate((4, 2, 2))]
    table = torch.arange(2, device=DEV, dtype=torch.int32).view(2, 1)
    pos = torch.full((T,), 3, dtype=torch.int32, device=DEV)
    out = []
    for q, k, v in (views, [x.reshape(x.numel()).clone().view(x.shape) for x in views]):
        cache = PagedKVCache.empty(2, 2, page, D)
        rotated = ops.append_kv(cache, q, k, v, table, pos, None)
        out.append((rotated, ops.paged_attention(cache, q, table, pos + 1), cache.k, cache.v))
    for a, b in zip(*out):
        assert torch.equal(a, b)
    assert out[0][0].shape == (T, 4, D) and ops.device_status() == 0


@pytest.mark.parametrize("shape", [(1, 2, 16, 64), (4, 1, 16, 64), (4, 2, 1, 64), (1, 1, 1, 64)])
def test_cache_axes_of_one(shape):
    """The stride of an axis of one is no reason to refuse a cache, nor to tell keys and values apart."""
    k, v = rand(shape, 1), rand(shape, 2)
    strides = lambda odd: [s if n > 1 else odd for s, n in zip(k.stride(), shape)]  # noqa: E731
    want, got = PagedKVCache(k.clone(), v.clone()), PagedKVCache(k.as_strided(shape, strides(13)), v.as_strided(shape, strides(7)))
    q = rand((1, 4, 64), 3)
    x = rand((1, shape[1], 64), 4)
    table = torch.zeros((1, 1), dtype=torch.int32, device=DEV)
    at = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = [(ops.append_kv(c, q, x, x, table, at, None), ops.paged_attention(c, q, table, at + 1), c.k, c.v) for c in (want, got)]
    for a, b in zip(*out):
        assert torch.equal(a, b)
    with pytest.raises(ValueError):
        PagedKVCache(rand((4, 2, 16, 64), 1).transpose(1, 2), rand((4, 16, 2, 64), 1))


@pytest.mark.parametrize("Hq,Hkv,D,T", [(4, 2, 64, 300), (8, 4, 128, 300), (2, 3, 256, 300), (2, 24, 128, 2400)])
def test_append_codes_equal_the_definition(Hq, Hkv, D, T):
    """An 8-bit cache holds e4m3(value / scale), the quotient in fp32, code for code; the last size has several heads a lane.
    Keys are neither normed nor rotated here."""
    page = 16
    cache = PagedKVCache.empty(-(-T // page), Hkv, page, D, F8, *(
        0.005 + 0.1 * torch.rand(Hkv, generator=torch.Generator(device=DEV).manual_seed(i), device=DEV) for i in (1, 2)))
    q, k, v = rand((T, Hq, D), 3), rand((T, Hkv, D), 4), rand((T, Hkv, D), 5)
    table = torch.arange(-(-T // page), device=DEV, dtype=torch.int32)[None]
    pos = torch.arange(T, device=DEV, dtype=torch.int32)
    ops.append_kv(cache, q, k, v, table, pos, None, rows=torch.zeros_like(pos))
    for c, x, s in ((cache.k, k, cache.k_scale), (cache.v, v, cache.v_scale)):
        got = c.view(torch.uint8).transpose(1, 2).flatten(0, 1)[:T]
        want = (x.float() / s[:, None]).clamp(-448, 448).to(F8).view(torch.uint8)
        assert torch.equal(got, want), int((got != want).sum())


def test_append_with_the_smallest_scales():
    """Zeros stay zeros and values saturate, at scales whose reciprocal is no fp32 number."""
    scale = torch.tensor([1e-39, 1e-45], device=DEV)
    cache = PagedKVCache.empty(1, 2, 16, 64, F8, scale, scale)
    k = torch.zeros((1, 2, 64), dtype=BF, device=DEV)
    k[0, :, 0] = 1.0
    table = torch.zeros((1, 1), dtype=torch.int32, device=DEV)
    ops.append_kv(cache, k, k, -k, table, table[0], None)
    for c, top in ((cache.k, 448), (cache.v, -448)):
        got = c[0, :, 0].float()
        assert bool((got[:, 0] == top).all()) and bool((got[:, 1:] == 0).all())


def test_append_rounds_ties_to_even():
    """Values that are a middle of two e4m3 numbers times the scale: the quotient is that middle, and goes to the even one."""
    page, D, T = 16, 128, 64
    scale = torch.tensor([3.0, 5.0, 7.0, 0.625], device=DEV)  # three bits: the product with a middle's five is a bf16 value
    cache = PagedKVCache.empty(T // page, 4, page, D, F8, scale, scale)
    r = torch.Generator().manual_seed(1)
    middle = (2 * torch.randint(8, 16, (T, 4, D), generator=r) + 1) * 2.0 ** torch.randint(-8, 4, (T, 4, D), generator=r)
    v = (middle.to(DEV) * scale[:, None]).to(BF)
    assert torch.equal(v.double() / scale.double()[:, None], middle.to(DEV).double())
    table = torch.arange(T // page, device=DEV, dtype=torch.int32)[None]
    pos = torch.arange(T, device=DEV, dtype=torch.int32)
    ops.append_kv(cache, v, v, v, table, pos, None, rows=torch.zeros_like(pos))
    want = middle.to(F8).view(torch.uint8).to(DEV)
    for c in (cache.k, cache.v):
        got = c.view(torch.uint8).transpose(1, 2).flatten(0, 1)
        assert torch.equal(got, want), int((got != want).sum())
