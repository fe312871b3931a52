"""The paged attention's kernel for many rows (17 a sequence and more, 16-bit types, heads of 64 or 128) where numbers
leave the ordinary sizes: scores from 1e-8 to 1e5, scales that grow and fall from tile to tile or differ between the
groups and positions of one tile.

Results are compared element by element with the 64-bit definition.  The bound is the kernel's roundings, propagated:

* a score is a sum of products of exact 16-bit numbers in fp32 (2^-20 of the sum of their sizes is allowed for), with
  values of q below 2^-14 of the row's largest rounded to 2^-25 of it;
* a weight is rounded to 11 bits, below 2^-14 of float16's normal numbers to a fixed step: 2^-32 of softmax's largest weight,
  2^-30 of SiLU's bound on the scores;
* SiLU's tanh is off by 2^-11 of half the score;
* sums of weights times values in fp32 (2^-16 of the sum of their sizes), one rounding of the result.
"""

import pytest
import torch

import generative_recommenders_b200 as G
from oracle import paged_oracle as P
from oracle.hstu_oracle import valid_attn_mask

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}    # one rounding of a result
SMALL = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}  # and below the normal numbers


def make_cache(lengths, H, d, page, k_exp=None, v_exp=None, seed=0, signs=False):
    """Random codes; scales of 0.2 to 0.5 (with ``signs`` -0.2 to -0.5 as well, and code 0) times 2^exp, ``exp(b, position, group)``
    whole numbers that broadcast."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lengths]
    order = torch.randperm(sum(need) + 2, generator=g)
    table = torch.full((len(lengths), max(need)), -1, dtype=torch.int32)
    pool = torch.full((sum(need) + 2, H, G.PagedKVCache.page_bytes(page, d)), 255, dtype=torch.uint8)
    codes, groups = page * d // 2, d // 64
    at = 0
    for b, n in enumerate(lengths):
        for i in range(need[b]):
            p = int(order[at])
            at += 1
            table[b, i] = p
            m = min(page, n - i * page)
            pos = torch.arange(i * page, i * page + m)[:, None]
            for kv, exp in enumerate((k_exp, v_exp)):
                x = torch.randint(0 if signs else 1, 16, (H, m, d), generator=g)
                pool[p, :, kv * codes:kv * codes + m * d // 2] = (x[..., 0::2] | x[..., 1::2] << 4).to(torch.uint8).flatten(1)
                s = torch.rand(H, m, groups, generator=g, dtype=torch.float64) * 0.3 + 0.2
                if signs:
                    s = s * (torch.randint(0, 2, s.shape, generator=g) * 2 - 1)
                if exp is not None:
                    s = s * 2.0 ** exp(b, pos, torch.arange(groups)[None]).double()
                raw = s.bfloat16().flatten(1).contiguous().view(torch.uint8)
                first = 2 * codes + kv * page * 2 * groups
                pool[p, :, first:first + raw.shape[1]] = raw
    return G.PagedKVCache(pool.to(DEV), page, d), table.to(DEV)


def offsets_of(counts):
    return torch.tensor([0] + list(counts)).cumsum(0).to(DEV)


def definition(q, k, v, length, targets, window, context, alpha, scale, softmax, dtype):
    """``(out, bound) [n, H, d]`` of the last n rows; what is NaN in the cache counts where it is seen."""
    n, H, d = q.shape
    group = H // k.shape[1]
    mask = valid_attn_mask(length, targets, True, window, context, 0).bool()[length - n:].to(DEV)
    q = q.double().transpose(0, 1)
    k, v = (x.to(DEV).repeat_interleave(group, 1).transpose(0, 1) for x in (k, v))
    s = q @ k.transpose(1, 2) * alpha
    sizes = q.abs() @ k.abs().transpose(1, 2) * abs(alpha)
    off = 2.0 ** -20 * sizes + 2.0 ** -24 * abs(alpha) * q.abs().amax(-1, keepdim=True) * k.abs().sum(-1)[:, None]
    none = torch.zeros((), dtype=torch.float64, device=DEV)
    if softmax:
        w = torch.softmax(s.masked_fill(~mask, float("-inf")), -1)
        error = w * (2.0 ** -11 + torch.expm1(off)) + 2.0 ** -32 * w.amax(-1, keepdim=True)
        common = (w * torch.expm1(off)).sum(-1, keepdim=True) + 2.0 ** -16
    else:
        w = torch.where(mask, s * torch.sigmoid(s), none)
        most = abs(alpha) * d * q.abs().amax(-1, keepdim=True) * k.abs().amax((1, 2), keepdim=True)
        error = 2.0 ** -11 * (w.abs() + s.abs() / 2) + 1.1 * off + 2.0 ** -30 * most
        common = none
        w, error = w * scale, error * scale
    error = torch.where(mask, error + 2.0 ** -16 * w.abs(), none)
    seen = mask.any(0)[:, None]
    clean = torch.where(seen & ~torch.isnan(v), v, none)
    out = w @ clean
    bound = error @ clean.abs() + out.abs() * (common + UNIT[dtype]) + SMALL[dtype]
    lost = mask.double() @ torch.isnan(torch.where(seen, v, none)).double() > 0
    out = torch.where(lost, torch.full_like(out, float("nan")), out)
    return out.transpose(0, 1), bound.transpose(0, 1)


def check(cache, table, lengths, new, Hq, dtype, softmax, targets=None, window=0, context=0, alpha=None, scale=1.0, seed=0):
    d = cache.head_dim
    alpha = d ** -0.5 if alpha is None else alpha
    q = torch.randn(sum(new), Hq, d, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)
    nt = None if targets is None else torch.tensor(targets, device=DEV)
    got = G.paged_mha(1, alpha, q, cache, table, torch.tensor(lengths, device=DEV), offsets_of(new), nt, window, context,
                      "softmax" if softmax else "silu", scale).double()
    at = 0
    for b, (n, m) in enumerate(zip(lengths, new)):
        k, v, _, _ = P.read_rows(cache, table[b].cpu(), n)
        out, bound = definition(q[at:at + m], k, v, n, 0 if targets is None else targets[b], window, context, alpha, scale,
                                softmax, dtype)
        x = got[at:at + m]
        at += m
        assert torch.equal(torch.isnan(x), torch.isnan(out)), b
        x, out = x.nan_to_num(0.0), out.nan_to_num(0.0)
        assert torch.isfinite(x).all(), b
        worst = float(((x - out).abs() / bound).max())
        assert worst <= 1, (b, worst)


ROWS = [([300, 150, 40], [40, 20, 33]), ([700, 420, 17], [300, 129, 17])]   # one block of rows, and two


@pytest.mark.parametrize("size", [1e-8, 1e-6, 1e-3, 1.0, 30.0, 1e3, 1e5])
@pytest.mark.parametrize("softmax", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lengths,new", ROWS)
def test_scores_of_any_size(lengths, new, dtype, softmax, size):
    cache, table = make_cache(lengths, 2, 128, 64, seed=3)
    for alpha in (size, -size):
        check(cache, table, lengths, new, 4, dtype, softmax, alpha=alpha * 128 ** -0.5, scale=0.01 / size)


@pytest.mark.parametrize("step", [1, 4, 8, 20, -1, -4, -8, -20])
@pytest.mark.parametrize("softmax", [False, True])
@pytest.mark.parametrize("window", [0, 100])
@pytest.mark.parametrize("lengths,new", ROWS)
def test_values_that_grow_and_fall_from_tile_to_tile(lengths, new, window, softmax, step):
    """V's scales change by 2^step every 128 positions; a window keeps rows from tiles that others of their block see."""
    def exp(b, pos, group):
        return (pos // 128) * step - (0 if step < 0 else 5 * step) + 0 * group

    for d in (64, 128):
        cache, table = make_cache(lengths, 2, d, 32, v_exp=exp, seed=d)
        check(cache, table, lengths, new, 2, torch.bfloat16, softmax, window=window)
        # scores of some size, so that weights and values are large together
        check(cache, table, lengths, new, 2, torch.bfloat16, softmax, window=window, alpha=2.0)


@pytest.mark.parametrize("step", [3, 9, -3, -9])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lengths,new", ROWS)
def test_keys_that_grow_and_fall_from_tile_to_tile(lengths, new, dtype, step):
    def exp(b, pos, group):
        return (pos // 128) * step - (0 if step < 0 else 5 * step) + 0 * group

    cache, table = make_cache(lengths, 2, 64, 16, k_exp=exp, seed=4)
    for window in (0, 100):
        check(cache, table, lengths, new, 4, dtype, False, window=window, scale=0.1)


@pytest.mark.parametrize("softmax", [False, True])
@pytest.mark.parametrize("lengths,new", ROWS)
def test_tiles_of_zeros_and_tiny_values(lengths, new, softmax):
    """The first 128 positions hold zeros, the others numbers around 2^-40."""
    def exp(b, pos, group):
        return torch.where(pos < 128, -1000, -40) + 0 * group

    cache, table = make_cache(lengths, 1, 128, 64, v_exp=exp, seed=6)
    for window in (0, 60):
        check(cache, table, lengths, new, 2, torch.bfloat16, softmax, window=window)


SPREAD = {
    # exponents of the scales within a tile
    "first group small": lambda b, pos, group: -20 * (group == 0) + 0 * pos,
    "second group small": lambda b, pos, group: -20 * (group == 1) + 0 * pos,
    "positions": lambda b, pos, group: -((pos * 7919 + b) % 21) + 0 * group,
    "one large": lambda b, pos, group: 20 * (pos % 128 == 77) - 10 + 0 * group,
    "groups and positions": lambda b, pos, group: -((pos * 31 + group * 11) % 21),
}


@pytest.mark.parametrize("spread", sorted(SPREAD))
@pytest.mark.parametrize("softmax", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lengths,new", ROWS)
def test_scales_far_apart_within_a_tile(lengths, new, dtype, softmax, spread):
    """Up to 2^20 between the scales of a tile, in V and in K: of positions that a row need not see (a window of a few,
    candidates that see none of each other) and of the groups, which are columns of their own."""
    exp = SPREAD[spread]
    targets = [n // 2 for n in new]
    for k_exp, v_exp in ((None, exp), (exp, None)):
        cache, table = make_cache(lengths, 2, 128, 64, k_exp, v_exp, seed=7)
        for nt, window in ((None, 0), (None, 3), (targets, 0), (targets, 3)):
            check(cache, table, lengths, new, 2, dtype, softmax, nt, window)


@pytest.mark.parametrize("softmax", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lengths,new", ROWS + [([300, 150, 40], [5, 2, 9])])
def test_values_that_are_no_numbers(lengths, new, dtype, softmax):
    """A group of V that is NaN makes that group's columns NaN of the rows that see it, and nothing else."""
    cache, table = make_cache(lengths, 2, 128, 64, seed=8)
    v = torch.randn(len(lengths), 2, 128, device=DEV)
    v[0, 0, 3] = float("inf")        # head 0, first group, of position 250
    v[1, 1, 100] = float("nan")      # head 1, second group, of position 140
    v[2, 0, 5] = v[2, 0, 127] = float("nan")   # both, of the last position
    at = torch.tensor([250, 140, lengths[2] - 1], device=DEV)
    G.append_paged_kv(cache, v.nan_to_num(1.0, 1.0), v, table, at, offsets_of([1] * 3))
    for targets, window in ((None, 0), (None, 20), ([n // 2 for n in new], 0)):
        check(cache, table, lengths, new, 4, dtype, softmax, targets, window)


@pytest.mark.parametrize("softmax", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [40, 140])
def test_positions_without_a_page(rows, dtype, softmax):
    """Rows that see a position past the table or on a page that is none are NaN, the others as ever."""
    lengths = [300, 270, 150]
    cache, table = make_cache(lengths, 2, 64, 16, seed=2)
    bad = table.clone()
    bad[0, 12] = -1                       # positions 192 ..
    bad[1, 16] = cache.num_pages + 5      # 256 ..
    q = torch.randn(3 * rows, 4, 64, generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
    most = 16 * table.shape[1]
    for window in (0, 30):
        good, out = (G.paged_mha(512, 0.1, q, cache, t, torch.tensor(n, device=DEV), offsets_of([rows] * 3),
                                 max_attn_len=window, activation="softmax" if softmax else "silu").view(3, rows, 4, 64)
                     for t, n in ((table, lengths), (bad, [300, 270, most + 3])))
        nan = torch.isnan(out).flatten(2)
        assert torch.equal(nan.any(2), nan.all(2))
        pos = torch.tensor([300, 270, most + 3])[:, None] - rows + torch.arange(rows)
        start = (pos - window).clamp(min=0) if window else torch.zeros_like(pos)
        first, last = torch.tensor([[192, 208], [256, 272], [150, 1000]]).unbind(1)   # (from 150 on: never written, ones)
        assert torch.equal(nan.all(2).cpu(), (pos >= first[:, None]) & (start < last[:, None]))
        same = ~nan.all(2)
        same[2] = False
        assert float((out[same].double() - good[same].double()).norm()) <= 2 * UNIT[dtype] * float(good[same].double().norm())


@pytest.mark.parametrize("softmax", [False, True])
@pytest.mark.parametrize("lengths,new", ROWS + [([300, 150, 40], [5, 2, 9])])
def test_negative_scales(lengths, new, softmax):
    """A cache that another program has filled: a scale is any finite bfloat16, a code any of 16."""
    for d in (64, 128):
        cache, table = make_cache(lengths, 2, d, 64, seed=9, signs=True)
        check(cache, table, lengths, new, 4, torch.bfloat16, softmax)
        top = cache.pages.clone()
        at, groups = 64 * d, d // 64      # (of a head of a page: codes, then scales)
        top[..., at:] = torch.tensor([0x7f, 0x3f], dtype=torch.uint8, device=DEV).repeat(2 * 64 * groups)   # 0.99609375
        check(G.PagedKVCache(top, 64, d), table, lengths, new, 4, torch.float16, softmax)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [1, 12, 40, 300])
@pytest.mark.parametrize("length", [1025, 10 ** 6 + 1, 2 ** 31 - 1])
def test_lengths_far_past_the_table(length, rows, dtype):
    """What is past the table costs nothing: the rows that see some of it are NaN, without a walk to a length that no
    cache has."""
    lengths = [1000, 1000, 700]
    cache, table = make_cache(lengths, 2, 64, 64, seed=4)
    q = torch.randn(3 * rows, 4, 64, generator=torch.Generator().manual_seed(2)).to(dtype).to(DEV)
    for act in ("silu", "softmax"):
        good, out = (G.paged_mha(1024, 0.1, q, cache, table, torch.tensor(n, device=DEV), offsets_of([rows] * 3),
                                 activation=act).double().view(3, rows, 4, 64) for n in (lengths, [1000, length, 700]))
        first = max(0, 1024 - length + rows)   # rows of the second sequence before the table's end see what they saw
        assert torch.isnan(out[1, first:]).all()
        for b in (0, 2):
            assert float((out[b] - good[b]).norm()) <= 2 * UNIT.get(dtype, 1e-5) * float(good[b].norm())
    # a table of no pages at all
    none = torch.zeros(1, 0, dtype=torch.int32, device=DEV)
    x = G.paged_mha(1024, 0.1, q[:rows], cache, none, torch.tensor([length], device=DEV), offsets_of([rows]))
    assert torch.isnan(x).all()
