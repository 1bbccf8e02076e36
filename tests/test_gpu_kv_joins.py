"""What the attention over a paged cache puts together from its parts (waves of a
workgroup, workgroups of a sequence): values that are not finite stay in the result
however small their part's weight is, and no part is lost or counted twice."""

from __future__ import annotations

import pytest
import torch

import kv_reference as ref
from test_gpu_kv_cache import bits, filled, gen, to

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
INF, NAN = float("inf"), float("nan")
TILE, WAVE = 128, 32  # positions that a workgroup, and a wave of it, take at a time


def places(cache, table, b, positions):
    p = torch.as_tensor(positions)
    return table[b, p // cache.key.shape[2]].long(), p % cache.key.shape[2]


def scored(g, lengths, heads, kv_heads, dim, fp8, scores):
    """A cache, a table and queries whose scores at scale 1 are those of ``scores``
    ({sequence: [length]}): the queries' first dimension is 1 and a key is its score
    there and 0 elsewhere."""
    cache, table = filled(g, lengths, kv_heads, 16, dim, fp8)
    for b, s in scores.items():
        page, slot = places(cache, table, b, range(lengths[b]))
        bits(cache.key)[page, :, slot] = 0
        if fp8:
            bits(cache.key)[page, :, slot, 0] = torch.where(s < 0, 0xB8, 0x38).to(torch.uint8)[:, None]  # -1, 1
            cache.key_scales[page, :, slot] = s.abs()[:, None]
        else:
            cache.key[page, :, slot, 0] = s.to(torch.bfloat16)[:, None]
    q = torch.zeros(len(lengths), heads, dim, dtype=torch.bfloat16)
    q[:, :, 0] = 1
    return cache, table, q


def attend(ext, cache, table, q, lengths):
    n32 = torch.tensor(lengths, dtype=torch.int32)
    out = ext.paged_attention(q.to(DEV), to(cache), table.to(DEV), n32.to(DEV), scale=1.0)
    torch.cuda.synchronize()
    return out.float().cpu()


# One workgroup's; in parts that a wave joins, and that a workgroup joins.
SPREAD = {"whole": 500, "few": 1300, "many": 20000}


@pytest.mark.parametrize("heads", [2, 24])  # one product a weight, and two
@pytest.mark.parametrize("dim", [64, 128, 192])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("spread", list(SPREAD))
@pytest.mark.parametrize("low", [WAVE, TILE])  # whose scores are far below all others': a wave's of every tile, a tile's
def test_what_is_not_finite_stays(hip_ext, spread, low, fp8, dim, heads):
    """A NaN key, a NaN value, an infinite value, and a NaN value behind a score of -inf,
    at a position whose neighbours' scores lie 200 below all others (a factor that
    underflows to 0)."""
    print(f"[case] not finite {spread} {low} {fp8} {dim} {heads}", flush=True)
    n = SPREAD[spread]
    at = 2 * TILE + 2 * WAVE + 5
    p = torch.arange(n)
    s = torch.where(p // TILE == at // TILE if low == TILE else p % TILE // WAVE == at % TILE // WAVE, -200.0, 0.0)
    cache, table, q = scored(gen(dim), [n, 40], heads, 2, dim, fp8, {0: s, 1: torch.zeros(40)})
    page, slot = places(cache, table, 0, [at])

    def with_(fill, value, score=None):
        k = to(cache, "cpu")._replace(**{f: getattr(cache, f).clone() for f in ("key", "value")},
                                      **({f: getattr(cache, f).clone() for f in ("key_scales", "value_scales")} if fp8 else {}))
        if score is not None:
            if fp8:
                k.key_scales[page, :, slot] = abs(score)  # (the code is -1)
            else:
                k.key[page, :, slot, 0] = score
        if fill == "key":
            (k.key_scales if fp8 else k.key)[page, :, slot] = value
        elif fp8 and value != value:
            bits(k.value)[page, :, slot, 3] = 0x7F
        elif fp8:
            k.value_scales[page, :, slot] = value
        else:
            k.value[page, :, slot, 3] = value
        out = attend(hip_ext, k, table, q, [n, 40])
        assert out[1].isfinite().all()
        return out[0]

    assert attend(hip_ext, cache, table, q, [n, 40]).isfinite().all()
    assert with_("key", NAN).isnan().all()
    for score in (None, -INF):
        got = with_("value", NAN, score)
        assert got[:, 3].isnan().all() and got[:, 4:].isfinite().all()
    got = with_("value", INF)
    assert not got[:, 3].isfinite().any() and (fp8 or got[:, 4:].isfinite().all())


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("n", [100, 3 * TILE + 4, 10 * TILE + 4, 156 * TILE + 4])
def test_a_part_of_nothing_but_nan(hip_ext, n, fp8):
    """The last four positions, which are their wave's only ones, have NaN keys; all
    other scores are 200 (a part without a finite score counts as one whose maximum is 0)."""
    print(f"[case] nan part {n} {fp8}", flush=True)
    cache, table, q = scored(gen(n), [n, 40], 4, 2, 64, fp8, {0: torch.full((n,), 200.0), 1: torch.zeros(40)})
    page, slot = places(cache, table, 0, range(n - 4, n))
    (cache.key_scales if fp8 else cache.key)[page, :, slot] = NAN
    got = attend(hip_ext, cache, table, q, [n, 40])
    assert got[0].isnan().all() and got[1].isfinite().all()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("n", [100, 3 * TILE + 4, 10 * TILE + 4, 156 * TILE + 4])
def test_a_part_of_scores_without_weight(hip_ext, n, fp8):
    """Scores of -inf in a part of their own take no weight, and a sequence of nothing else is NaN."""
    print(f"[case] -inf part {n} {fp8}", flush=True)
    s = torch.zeros(n)
    s[n - 4:] = -INF
    cache, table, q = scored(gen(n), [n, 40], 4, 2, 64, fp8, {0: s, 1: torch.full((40,), -INF)})
    if not fp8:  # (a query's 0 times an infinity would be a NaN; here only the first dimension is one)
        assert cache.key[..., 1:].isinf().sum() == 0
    got = attend(hip_ext, cache, table, q, [n, 40])
    assert got[1].isnan().all()
    v, _ = ref.position_rows(cache.value, cache.value_scales, table[0], torch.arange(n - 4))
    want = v.mean(0).repeat_interleave(2, 0)
    # (n FP32 sums and the two numbers of a weight beside the output's rounding)
    off = (2.0 ** -16 + 4 * n * ref.U) * v.abs().mean(0).repeat_interleave(2, 0)
    assert ((got[0].double() - want).abs() <= off * (1 + ref.BF16) + ref.BF16 * want.abs()).all()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("n", [100, 3 * TILE + 4, 10 * TILE + 4, 156 * TILE + 4])
def test_an_infinite_score(hip_ext, n, fp8):
    """One score of +inf: NaN (inf - inf), wherever it lies."""
    print(f"[case] +inf {n} {fp8}", flush=True)
    for at in (0, n // 2, n - 1):
        s = torch.zeros(n)
        s[at] = INF
        cache, table, q = scored(gen(n), [n, 40], 4, 2, 64, fp8, {0: s, 1: torch.zeros(40)})
        got = attend(hip_ext, cache, table, q, [n, 40])
        assert got[0].isnan().all() and got[1].isfinite().all()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("heads", [32, 36])
def test_what_is_not_finite_stays_among_many_sequences(hip_ext, heads, fp8):
    """The same where parts are joined column by column (more heads than the card has waves)."""
    print(f"[case] not finite, columns {heads} {fp8}", flush=True)
    n, at, lengths = 3000, 1500, [40] * 150 + [3000] + [40] * 150
    s = torch.where(torch.arange(n) // TILE == at // TILE, -200.0, 0.0)
    zeros = {b: torch.zeros(m) for b, m in enumerate(lengths)}
    for fill, where in (("key", (0,)), ("value", (3,))):
        cache, table, q = scored(gen(heads), lengths, heads, 2, 64, fp8, {**zeros, 150: s})
        page, slot = places(cache, table, 150, [at])
        if fp8:
            bits(getattr(cache, fill))[page, :, slot, where[0]] = 0x7F
        else:
            getattr(cache, fill)[page, :, slot, where[0]] = NAN
        got = attend(hip_ext, cache, table, q, lengths)
        assert got[150, :, 3].isnan().all() and got[150, :, 4:].isnan().all().item() == (fill == "key")
        assert got[:150].isfinite().all() and got[151:].isfinite().all()


def test_many_sequences_cost_no_more_each(hip_ext):
    """Four times as many sequences in a wide table take some four times as long, not sixteen."""
    print("[case] cost of many sequences", flush=True)
    cache = hip_ext.new_kv_cache(8, 1, 16, 64, device=DEV)
    took = []
    for batch in (16384, 65536):
        table = torch.arange(72, dtype=torch.int32, device=DEV).remainder(8).expand(batch, -1).contiguous()
        lengths = torch.full((batch,), 50, dtype=torch.int32, device=DEV)
        query = torch.ones(batch, 8, 64, dtype=torch.bfloat16, device=DEV)
        times = []
        for _ in range(4):
            start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            start.record()
            hip_ext.paged_attention(query, cache, table, lengths)
            end.record()
            torch.cuda.synchronize()
            times.append(start.elapsed_time(end))
        took.append(min(times))
    assert took[1] < 8 * took[0], took


# Lengths that go over columns of one and of several tiles, joins by waves and by
# workgroups, more sequences than columns.
MARKED = [
    (4, 4, 128, [20000], None), (8, 1, 64, [40001], None), (2, 1, 256, [9999, 3], None), (16, 4, 128, [1, 0, 8191, 30, 4097], None),
    (3, 3, 80, [1000 + 38 * i for i in range(70)], None), (32, 2, 96, [5000, 77], None), (1, 1, 64, [65001], None),
    (1, 1, 256, [131071], None), (20, 1, 128, [60001, 700], None), (4, 2, 64, [300 * i for i in range(17)], None),
    (16, 16, 48, [(211 * i) % 1500 for i in range(40)], None), (2, 1, 64, [9000, 700, 20001], 5003),
    (6, 2, 96, [(977 * i) % 4000 for i in range(33)], 1234),
    # (more heads than waves: joined column by column)
    (64, 4, 64, [(211 * i) % 1500 for i in range(140)], None), (40, 40, 16, [(101 * i) % 1100 for i in range(220)], None),
    (160, 10, 80, [0] * 30 + [20000] + [5] * 30 + [1], None), (256, 16, 144, [900] * 17 + [7000] * 17, 3000),
    (288, 288, 16, [1500, 0, 30] * 10, None),
]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim,lengths,window", MARKED)
def test_every_position_counts_once(hip_ext, heads, kv_heads, dim, lengths, window, fp8):
    """Queries of 0 weigh all positions alike, and the values of 16 positions are 1 in one
    dimension, which goes by their place, sequence and head. An output is then the part of
    the positions that mark its dimension: whole numbers below 2^24 are exact in FP32, so
    that the quotient is off by the reciprocal's, the product's and the output's rounding.
    Sixteen positions lost or doubled change it by dim / (positions / 16), four such
    roundings or more."""
    print(f"[case] marks {heads} {kv_heads} {dim} {lengths[:5]} {window} {fp8}", flush=True)
    longest = max(min(n, window or n) for n in lengths)
    assert 16 * dim >= 4 * ref.BF16 * longest
    g = gen(dim + heads)
    cache, table = filled(g, lengths, kv_heads, 16, dim, fp8)
    want = torch.zeros(len(lengths), kv_heads, dim, dtype=torch.float64)
    for b, n in enumerate(lengths):
        if n == 0:
            continue
        p = torch.arange(n)
        mark = (p[:, None] // 16 + 7 * b + 3 * torch.arange(kv_heads)) % dim  # [positions, kv_heads]
        rows = torch.nn.functional.one_hot(mark, dim)
        page, slot = places(cache, table, b, p)
        if fp8:
            bits(cache.value)[page, :, slot] = (0x38 * rows).to(torch.uint8)
            cache.value_scales[page, :, slot] = 0.5
        else:
            cache.value[page, :, slot] = (0.5 * rows).to(torch.bfloat16)
        first = max(0, n - window) if window else 0
        want[b] = rows[first:].sum(0).double() / (2 * (n - first))
    n32 = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    q = torch.zeros(len(lengths), heads, dim, dtype=torch.bfloat16, device=DEV)
    got = hip_ext.paged_attention(q, to(cache), table.to(DEV), n32, window=window).double().cpu()
    want = want.repeat_interleave(heads // kv_heads, 1)
    assert ((got - want).abs() <= (ref.BF16 + 4 * ref.U) * want).all()
