"""The paged key-value cache on the device: rows put in, rows read back, and the
attention of one new token, against plain forms in 64 bits. Places that no call may
read hold NaN, and places that no call may write are compared bit by bit."""

from __future__ import annotations

import pytest
import torch

import kv_reference as ref
from uma_qmoe_amd.native_backend import KVCache

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F8 = torch.float8_e4m3fn


def gen(seed):
    return torch.Generator().manual_seed(seed)


def normal(g, *shape):
    return torch.randn(*shape, generator=g)


def poisoned(pages, kv_heads, page_size, dim, fp8):
    """A cache of NaN (codes and scales)."""
    shape = (pages, kv_heads, page_size, dim)
    if fp8:
        codes = [torch.full(shape, 0x7F, dtype=torch.uint8).view(F8) for _ in range(2)]
        return KVCache(*codes, *(torch.full(shape[:3], float("nan")) for _ in range(2)))
    return KVCache(*(torch.full(shape, float("nan"), dtype=torch.bfloat16) for _ in range(2)))


def bits(t):
    return t.view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()])


def make_table(g, lengths, page_size, spare=3, width=None):
    """A table of shuffled pages; entries behind a sequence's end name pages all the
    same (which must not be looked at), one in three of them none."""
    used = [-(-max(n, 0) // page_size) for n in lengths]
    pages = sum(used) + spare
    free = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.randint(0, pages, (len(lengths), width or max([1, *used])), generator=g, dtype=torch.int32)
    table[torch.rand(table.shape, generator=g) < 0.33] = -7
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = free[at:at + n]
        at += n
    return table, pages


def filled(g, lengths, kv_heads, page_size, dim, fp8, spare=3, width=None, scale=1.0):
    """A cache (CPU) whose sequences hold normal values and everything else NaN, and its table."""
    table, pages = make_table(g, lengths, page_size, spare, width)
    cache = poisoned(pages, kv_heads, page_size, dim, fp8)
    for b, n in enumerate(lengths):
        if n <= 0:
            continue
        p = torch.arange(n)
        page, slot = table[b, p // page_size].long(), p % page_size
        for data, scales, s in ((cache.key, cache.key_scales, scale), (cache.value, cache.value_scales, 1.0)):
            rows = s * normal(g, n, kv_heads, dim) * torch.exp(0.5 * normal(g, n, kv_heads, 1))
            if fp8:
                rows, scales[page, :, slot] = ref.quantize(rows.to(torch.bfloat16).float())
            else:
                rows = rows.to(torch.bfloat16)
            bits(data)[page, :, slot] = bits(rows)
    return cache, table


def to(cache, device=DEV):
    return KVCache(*(None if t is None else t.to(device) for t in cache))


# ------------------------------------------------------------------ append --
def append_case(ext, g, kv_heads, page_size, dim, fp8, starts, counts, tokens, given=True, lay=None):
    batch = len(starts)
    ends = [max(0, s + min(c, tokens)) for s, c in zip(starts, counts)]
    table, pages = make_table(g, ends, page_size)
    before = poisoned(pages, kv_heads, page_size, dim, fp8)
    cache = to(before)
    rows = [normal(g, batch, kv_heads, tokens, dim).mul(10.0 ** (i - 1)).to(torch.bfloat16) for i in range(2)]
    new = [lay(r) if lay else r.to(DEV) for r in rows]
    c32 = torch.tensor(counts, dtype=torch.int32, device=DEV) if given else None
    got = ext.kv_append(cache, *new, table.to(DEV), torch.tensor(starts, dtype=torch.int32, device=DEV), c32)
    assert got is cache
    torch.cuda.synchronize()
    check_append(before, to(cache, "cpu"), rows, table, starts, counts if given else [tokens] * batch)


def check_append(before, after, rows, table, starts, counts):
    page_size, tokens = before.key.shape[2], rows[0].shape[2]
    written = torch.zeros(before.key.shape[0], page_size, dtype=torch.bool)
    for b, (s, c) in enumerate(zip(starts, counts)):
        j = torch.arange(max(0, min(c, tokens)))
        p = s + j
        j, p = j[(p >= 0) & (p < table.shape[1] * page_size)], p[(p >= 0) & (p < table.shape[1] * page_size)]
        page = table[b, p // page_size].long()
        there = (page >= 0) & (page < before.key.shape[0])
        j, page, slot = j[there], page[there], (p % page_size)[there]
        written[page, slot] = True
        for data, scales, new in ((after.key, after.key_scales, rows[0]), (after.value, after.value_scales, rows[1])):
            want = new[b, :, j].transpose(0, 1)  # [rows, kv_heads, dim]
            have = bits(data)[page, :, slot].view(data.dtype)
            if scales is None:
                assert torch.equal(bits(have), bits(want.contiguous()))
            else:
                ref.check_codes(have, scales[page, :, slot], want.double())
    left = ~written
    for a, z in zip(before, after):
        if a is not None:
            assert torch.equal(bits(a).transpose(1, 2)[left], bits(z).transpose(1, 2)[left]), "a place that was not written"


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("kv_heads,page_size,dim", [(1, 16, 16), (3, 16, 64), (4, 32, 80), (16, 16, 128), (2, 64, 192), (5, 256, 256), (7, 128, 112)])
def test_append(hip_ext, kv_heads, page_size, dim, fp8):
    print(f"[case] append {kv_heads} {page_size} {dim} {fp8}", flush=True)
    g = gen(dim + kv_heads)
    append_case(hip_ext, g, kv_heads, page_size, dim, fp8, [0, 5, page_size - 1, 300], [37, 1, 0, 300], 37)
    append_case(hip_ext, g, kv_heads, page_size, dim, fp8, [0], [1], 1)
    append_case(hip_ext, g, kv_heads, page_size, dim, fp8, [3, 200, 16], [0, 0, 0], 1, given=False)


@pytest.mark.parametrize("fp8", [False, True])
def test_append_drops_rows_without_a_place(hip_ext, fp8):
    """Negative positions, positions behind the table, table entries that name no page."""
    print(f"[case] append drops {fp8}", flush=True)
    g = gen(3)
    kv_heads, page_size, dim, tokens = 2, 16, 64, 50
    table = torch.tensor([[0, -1, 2], [3, 99, 4], [5, 6, 7], [-2147483648, 2147483647, 8], [9, 10, 11]], dtype=torch.int32)
    starts, counts = [0, -20, 30, 5, 2147483647], [50, 50, 50, 41, 50]
    before = poisoned(13, kv_heads, page_size, dim, fp8)
    cache = to(before)
    rows = [normal(g, 5, kv_heads, tokens, dim).to(torch.bfloat16) for _ in range(2)]
    hip_ext.kv_append(cache, *(r.to(DEV) for r in rows), table.to(DEV), torch.tensor(starts, dtype=torch.int32, device=DEV),
                      torch.tensor(counts, dtype=torch.int32, device=DEV))
    torch.cuda.synchronize()
    check_append(before, to(cache, "cpu"), rows, table, starts, counts)


def strided(r):
    """[batch, heads, tokens, dim] as a view of [batch, tokens, heads, dim] rows of a wider tensor."""
    wide = torch.full((*r.transpose(1, 2).shape[:3], r.shape[3] + 8), float("nan"), dtype=r.dtype, device=DEV)
    wide[..., :r.shape[3]] = r.transpose(1, 2).to(DEV)
    return wide[..., :r.shape[3]].transpose(1, 2)


def shifted(r):
    """The same values two bytes behind an aligned address."""
    flat = torch.empty(r.numel() + 1, dtype=r.dtype, device=DEV)[1:].view(r.shape)
    return flat.copy_(r)


def last_strided(r):
    """Elements of a row apart."""
    return torch.stack([r, torch.full_like(r, float("nan"))], -1).to(DEV)[..., 0]


@pytest.mark.parametrize("lay", [strided, shifted, last_strided])
@pytest.mark.parametrize("fp8", [False, True])
def test_append_of_any_strides(hip_ext, lay, fp8):
    print(f"[case] append strides {lay.__name__} {fp8}", flush=True)
    append_case(hip_ext, gen(4), 3, 16, 80, fp8, [0, 7], [21, 13], 21, lay=lay)


def test_append_of_one_row_for_every_token(hip_ext):
    print("[case] append expanded", flush=True)
    g = gen(5)
    row = normal(g, 2, 1, 1, 64).to(torch.bfloat16)
    table, pages = make_table(g, [20, 20], 16)
    before = poisoned(pages, 3, 16, 64, True)
    cache = to(before)
    new = row.to(DEV).expand(2, 3, 20, 64)
    hip_ext.kv_append(cache, new, new, table.to(DEV), torch.zeros(2, dtype=torch.int32, device=DEV))
    torch.cuda.synchronize()
    rows = row.expand(2, 3, 20, 64).contiguous()
    check_append(before, to(cache, "cpu"), [rows, rows], table, [0, 0], [20, 20])


def test_append_of_special_rows(hip_ext):
    """Zeros have scale 1; tiny rows the least scale; a row with a NaN or an
    infinity reads back as NaN, and changes no other."""
    print("[case] append special", flush=True)
    dim = 64
    rows = torch.zeros(1, 1, 6, dim, dtype=torch.bfloat16)
    rows[0, 0, 1] = 1e-38
    rows[0, 0, 2] = 3e38 * torch.linspace(-1, 1, dim)  # (linspace overflows between the two)
    rows[0, 0, 3, 5] = float("nan")
    rows[0, 0, 4, 7] = float("inf")
    rows[0, 0, 5] = torch.linspace(-1, 1, dim)
    cache = hip_ext.new_kv_cache(1, 1, 16, dim, fp8=True, device=DEV)
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    hip_ext.kv_append(cache, rows.to(DEV), rows.to(DEV), table, torch.zeros(1, dtype=torch.int32, device=DEV))
    for codes, scales in ((cache.key, cache.key_scales), (cache.value, cache.value_scales)):
        assert scales[0, 0, 0] == 1 and scales[0, 0, 1] == 2.0 ** -126
        for i in (0, 1, 2, 5):
            ref.check_codes(codes[0, 0, i].cpu(), scales[0, 0, i].cpu(), rows[0, 0, i].double())
        back = codes[0, 0].float() * scales[0, 0][:, None]
        assert back[3].isnan().all() and not back[4].isfinite().any()
        assert bits(codes)[0, 0, 6:].eq(0).all()


# -------------------------------------------------------------------- read --
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("kv_heads,page_size,dim", [(1, 16, 16), (4, 32, 80), (16, 16, 128), (3, 64, 48), (2, 128, 256), (3, 256, 208)])
def test_read(hip_ext, kv_heads, page_size, dim, fp8):
    print(f"[case] read {kv_heads} {page_size} {dim} {fp8}", flush=True)
    g = gen(dim)
    lengths = [0, 1, 17, 300, 255, 16]
    cache, table = filled(g, lengths, kv_heads, page_size, dim, fp8)
    table[3, 0] = -1  # a sequence with a hole
    given = torch.tensor([-5, 1, 17, 300, 255, 16], dtype=torch.int32)
    for most in (1, 300, 301, table.shape[1] * page_size + 9):
        got = hip_ext.kv_read(to(cache), table.to(DEV), given.to(DEV), most)
        torch.cuda.synchronize()
        for t, data, scales in zip(got, cache[:2], cache[2:]):
            assert t.shape == (len(lengths), kv_heads, most, dim) and t.dtype is torch.bfloat16
            for b, n in enumerate(lengths):
                rows, there = ref.position_rows(data, scales, table[b], torch.arange(min(n, most)))
                want = torch.where(there[:, None, None], rows, 0.0).transpose(0, 1)
                have = t[b].double().cpu()
                assert (have[:, n:] == 0).all()
                # (the product with the scale is rounded to FP32, then to BF16)
                assert ((have[:, :want.shape[1]] - want).abs() <= (ref.BF16 * (1 + ref.U) + ref.U) * want.abs() * fp8).all()


def test_read_of_nothing(hip_ext):
    print("[case] read nothing", flush=True)
    cache = hip_ext.new_kv_cache(2, 3, 16, 32, device=DEV)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    assert hip_ext.kv_read(cache, none.view(0, 4), none, 7)[0].shape == (0, 3, 7, 32)
    one = torch.full((1,), 9, dtype=torch.int32, device=DEV)
    assert hip_ext.kv_read(cache, one.view(1, 1), one, 0)[1].shape == (1, 3, 0, 32)
    key, value = hip_ext.kv_read(cache, torch.zeros(1, 0, dtype=torch.int32, device=DEV), one, 9)
    assert key.eq(0).all() and value.eq(0).all()


# --------------------------------------------------------------- attention --
def attend_case(ext, g, lengths, heads, kv_heads, page_size, dim, fp8, window=None, scale=None, given=None, query=None, **kw):
    cache, table = filled(g, lengths, kv_heads, page_size, dim, fp8, **kw)
    q = (2 * normal(g, len(lengths), heads, dim)).to(torch.bfloat16) if query is None else query
    n32 = torch.tensor(given or lengths, dtype=torch.int32)
    got = ext.paged_attention(q.to(DEV), to(cache), table.to(DEV), n32.to(DEV), scale=scale, window=window)
    torch.cuda.synchronize()
    assert got.shape == q.shape and got.dtype is torch.bfloat16
    ref.check_attention(got, q, cache, table, n32, dim ** -0.5 if scale is None else scale, window)
    return got, q, cache, table


LENGTHS = [0, 1, 2, 15, 16, 17, 31, 33, 127, 128, 129, 500]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("page_size", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 2, 64), (16, 16, 128), (14, 2, 80), (8, 1, 256)])
def test_attention(hip_ext, heads, kv_heads, dim, page_size, fp8):
    print(f"[case] attention {heads} {kv_heads} {dim} {page_size} {fp8}", flush=True)
    attend_case(hip_ext, gen(dim + page_size), LENGTHS, heads, kv_heads, page_size, dim, fp8)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dim", list(range(16, 257, 16)))
def test_attention_of_every_head_size(hip_ext, dim, fp8):
    print(f"[case] attention dim {dim} {fp8}", flush=True)
    attend_case(hip_ext, gen(dim), [1, 37, 200], 6, 2, 16, dim, fp8)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("group", [1, 2, 3, 7, 8, 9, 15, 16, 17, 33, 48])
def test_attention_of_shared_heads(hip_ext, group, fp8):
    print(f"[case] attention group {group} {fp8}", flush=True)
    attend_case(hip_ext, gen(group), [0, 45, 300], 2 * group, 2, 32, 128, fp8)


@pytest.mark.parametrize("window", [1, 2, 16, 31, 100, 499, 500, 1 << 40])
@pytest.mark.parametrize("fp8", [False, True])
def test_attention_in_a_window(hip_ext, window, fp8):
    """Places before the window hold NaN too."""
    print(f"[case] attention window {window} {fp8}", flush=True)
    g = gen(window % 1000)
    cache, table = filled(g, LENGTHS, 4, 32, 64, fp8)
    for b, n in enumerate(LENGTHS):
        p = torch.arange(max(0, n - window))
        page, slot = table[b, p // 32].long(), p % 32
        for t in cache:
            if t is not None:
                bits(t)[page, :, slot] = 0x7F if t.element_size() == 1 else 0x7FC0 if t.element_size() == 2 else 0x7FC00000
    q = normal(g, len(LENGTHS), 8, 64).to(torch.bfloat16)
    n32 = torch.tensor(LENGTHS, dtype=torch.int32)
    got = hip_ext.paged_attention(q.to(DEV), to(cache), table.to(DEV), n32.to(DEV), window=window)
    ref.check_attention(got, q, cache, table, n32, 64 ** -0.5, window)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim,lengths", [
    (4, 4, 128, [20000]), (8, 1, 64, [40001]), (2, 1, 256, [9999, 3]), (16, 4, 128, [1, 0, 8191, 30, 4097]),
    (3, 3, 80, [1000 + 37 * i for i in range(70)]), (32, 2, 96, [5000, 77]), (1, 1, 16, [65537])])
def test_attention_over_long_sequences(hip_ext, heads, kv_heads, dim, lengths, fp8):
    """Long enough for several workgroups to share a sequence; batches beyond a wave."""
    print(f"[case] attention long {heads} {kv_heads} {dim} {lengths[:5]} {fp8}", flush=True)
    attend_case(hip_ext, gen(heads), lengths, heads, kv_heads, 16, dim, fp8)


@pytest.mark.parametrize("lengths", [[200, 5, 300], [700, 5, 1300]])  # heads whole, and in parts
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("group", [2, 12])
@pytest.mark.parametrize("dim", [64, 48, 128, 80, 256, 192])
def test_every_kernel(hip_ext, dim, group, fp8, lengths):
    """Whole and ragged head sizes of each width, one and two products a weight, both types, both ways to deal out work."""
    print(f"[case] attention kernels {dim} {group} {fp8} {lengths}", flush=True)
    attend_case(hip_ext, gen(dim + group), lengths, 3 * group, 3, 32, dim, fp8)


@pytest.mark.parametrize("batch", [63, 64, 65, 129, 300])
def test_attention_of_many_sequences(hip_ext, batch):
    print(f"[case] attention batch {batch}", flush=True)
    attend_case(hip_ext, gen(batch), [(37 * i) % 71 for i in range(batch)], 2, 2, 16, 32, True)
    attend_case(hip_ext, gen(batch), [(37 * i) % 71 for i in range(batch)], 2, 2, 16, 32, True, width=40)
    attend_case(hip_ext, gen(batch), [(211 * i) % 900 for i in range(batch)], 2, 2, 16, 32, False)
    attend_case(hip_ext, gen(batch), [0] * (batch - 1) + [1500], 2, 1, 16, 32, False)
    attend_case(hip_ext, gen(batch), [1500] + [0] * (batch - 1), 2, 1, 16, 32, False)


@pytest.mark.parametrize("fp8", [False, True])
def test_attention_skips_pages_that_are_none(hip_ext, fp8):
    print(f"[case] attention holes {fp8}", flush=True)
    g = gen(11)
    lengths = [100, 64, 4000, 33, 40]
    cache, table = filled(g, lengths, 2, 16, 64, fp8)
    table[0, 2] = -1
    table[1, :4] = 1 << 30      # nothing left
    table[2, 0::3] = -2147483648
    table[3, 2] = cache.key.shape[0]
    table[4, 0] = 2147483647
    q = normal(g, 5, 6, 64).to(torch.bfloat16)
    n32 = torch.tensor(lengths, dtype=torch.int32)
    got = hip_ext.paged_attention(q.to(DEV), to(cache), table.to(DEV), n32.to(DEV))
    ref.check_attention(got, q, cache, table, n32, 0.125)
    assert got[1].eq(0).all()


def test_attention_clamps_lengths(hip_ext):
    """A length below 0 is 0, one beyond the table the table's."""
    print("[case] attention lengths", flush=True)
    attend_case(hip_ext, gen(12), [0, 64, 64, 5], 2, 1, 16, 32, False, given=[-3, 65, 2147483647, 5])
    attend_case(hip_ext, gen(12), [0, 640, 640, 5], 2, 1, 16, 32, True, given=[-2147483648, 10000, 2147483647, 5])


@pytest.mark.parametrize("window", [1, 128, 129, 130, 384, 385, 386, 387, 500])
def test_windows_over_long_tables(hip_ext, window):
    """Windows whose tiles are one workgroup's, and the first that are not, at every offset within a tile."""
    print(f"[case] attention window of a long table {window}", flush=True)
    attend_case(hip_ext, gen(window), [5000 + 37 * i for i in range(9)] + [0, 1, window, window + 1], 2, 1, 16, 32, True, window=window)


@pytest.mark.parametrize("window", [None, 896, 897, 898, 899])
@pytest.mark.parametrize("width", [64, 65])  # pages of 16: eight tiles, and the first page of a ninth
@pytest.mark.parametrize("batch,heads,kv_heads", [(7, 16, 16), (9, 16, 16), (18, 40, 4)])
def test_tables_of_eight_tiles(hip_ext, batch, heads, kv_heads, width, window):
    """Sequences of up to eight tiles are one workgroup's a head where there are many of them;
    fewer sequences, one page more and longer windows are in parts."""
    print(f"[case] attention eight tiles {batch} {heads} {kv_heads} {width} {window}", flush=True)
    most = 16 * width
    lengths = ([most, 0, 1, most - 1, 513, 640, 897] * 3)[:batch]
    lengths[-1] = 1023
    attend_case(hip_ext, gen(width + batch), lengths, heads, kv_heads, 16, 32, batch % 2 == 0, window=window, width=width + (0 if window is None else 300))


@pytest.mark.parametrize("scale", [1.0, -0.3, 0.0, 3.0])
def test_attention_of_a_scale(hip_ext, scale):
    print(f"[case] attention scale {scale}", flush=True)
    attend_case(hip_ext, gen(13), [1, 50, 700], 4, 2, 16, 64, False, scale=scale)


@pytest.mark.parametrize("fp8", [False, True])
def test_attention_of_large_scores(hip_ext, fp8):
    """Scores far apart: one weight is nearly 1, others underflow; the running maximum moves often."""
    print(f"[case] attention peaked {fp8}", flush=True)
    attend_case(hip_ext, gen(14), [300, 5000], 4, 2, 16, 128, fp8, scale=0.5)


def special(ext, fill, where, value, fp8=False, n=1000, dim=64):
    """Attention over keys ``where`` of which are ``value``, of positive queries."""
    g = gen(15)
    cache, table = filled(g, [n], 1, 16, dim, fp8)
    p = torch.tensor(where)
    page, slot = table[0, p // 16].long(), p % 16
    if fp8:
        getattr(cache, fill + "_scales")[page, :, slot] = value
        bits(getattr(cache, fill))[page, :, slot] = 0x38  # 1.0
    else:
        getattr(cache, fill)[page, :, slot] = value
    q = (0.1 + torch.rand(1, 2, dim, generator=g)).to(torch.bfloat16)
    n32 = torch.tensor([n], dtype=torch.int32)
    got = ext.paged_attention(q.to(DEV), to(cache), table.to(DEV), n32.to(DEV)).double().cpu()
    return got, q, cache, table, n32


@pytest.mark.parametrize("fp8", [False, True])
def test_attention_of_special_scores(hip_ext, fp8):
    print(f"[case] attention special {fp8}", flush=True)
    inf, nan = float("inf"), float("nan")
    # a score of -inf takes no weight (its sequence's other scores are finite)
    for where in ([0], [999], list(range(0, 128)), list(range(500, 1000)), list(range(1, 1000))):
        got, q, cache, table, n32 = special(hip_ext, "key", where, -inf, fp8)
        keep = torch.ones(1000, dtype=torch.bool)
        keep[where] = False
        k, _ = ref.position_rows(cache.key, cache.key_scales, table[0], torch.arange(1000))
        v, _ = ref.position_rows(cache.value, cache.value_scales, table[0], torch.arange(1000))
        s = (k[:, 0][:, None] * q[0].double()).sum(2)[keep] / 8
        want = (torch.softmax(s, 0)[..., None] * v[keep]).sum(0)
        assert ((got[0] - want).abs() <= 2 * ref.BF16 * want.abs() + 2e-4).all()
    assert special(hip_ext, "key", list(range(1000)), -inf, fp8)[0].isnan().all()  # 0 / 0
    for where in ([0], [640], [999], list(range(1000))):
        assert special(hip_ext, "key", where, nan, fp8)[0].isnan().all()
        assert special(hip_ext, "key", where, inf, fp8)[0].isnan().all()  # inf - inf
        assert special(hip_ext, "value", where, nan, fp8)[0].isnan().all()
        assert not special(hip_ext, "value", where, inf, fp8)[0].isfinite().any()


def test_attention_without_a_page(hip_ext):
    """Tables of no column, and no sequence."""
    print("[case] attention without pages", flush=True)
    cache = hip_ext.new_kv_cache(2, 2, 16, 64, device=DEV)
    q = torch.ones(3, 4, 64, dtype=torch.bfloat16, device=DEV)
    none = torch.zeros(3, 0, dtype=torch.int32, device=DEV)
    assert hip_ext.paged_attention(q, cache, none, torch.full((3,), 5, dtype=torch.int32, device=DEV)).eq(0).all()
    hip_ext.kv_append(cache, q[:, :2, None], q[:, :2, None], none, torch.zeros(3, dtype=torch.int32, device=DEV))
    assert cache.key.eq(0).all()
    assert hip_ext.paged_attention(q[:0], cache, none[:0], torch.zeros(0, dtype=torch.int32, device=DEV)).shape == (0, 4, 64)


def test_attention_takes_views(hip_ext):
    """A query, a table and lengths that are parts of larger tensors, a table by columns or for all sequences."""
    print("[case] attention views", flush=True)
    g = gen(16)
    lengths = [40, 0, 77]
    cache, table = filled(g, lengths, 2, 16, 32, True)
    q = normal(g, 3, 4, 32).to(torch.bfloat16)
    n32 = torch.tensor(lengths, dtype=torch.int32)
    kv = to(cache)
    want = hip_ext.paged_attention(q.to(DEV), kv, table.to(DEV), n32.to(DEV))
    ref.check_attention(want, q, cache, table, n32, 32 ** -0.5)
    wide = torch.full((3, table.shape[1] + 5), -1, dtype=torch.int32, device=DEV)
    wide[:, 2:2 + table.shape[1]] = table.to(DEV)
    for t in (wide[:, 2:2 + table.shape[1]], table.t().contiguous().to(DEV).t()):
        for x in (strided(q[:, :, None])[:, :, 0], shifted(q)):
            both = torch.stack([n32, n32 * 0 - 1], 1).to(DEV)[:, 0]
            assert torch.equal(hip_ext.paged_attention(x, kv, t, both), want)
    same = hip_ext.paged_attention(q.to(DEV), kv, table[2:].to(DEV).expand(3, -1), torch.tensor([77, 77, 77], dtype=torch.int32, device=DEV))
    ref.check_attention(same, q, cache, table[2:].expand(3, -1), torch.tensor([77] * 3), 32 ** -0.5)


def test_attention_is_the_same_each_time(hip_ext):
    print("[case] attention repeats", flush=True)
    got, q, cache, table = attend_case(hip_ext, gen(17), [30000, 5, 1200], 8, 2, 16, 128, True)
    n32 = torch.tensor([30000, 5, 1200], dtype=torch.int32, device=DEV)
    for _ in range(5):
        assert torch.equal(hip_ext.paged_attention(q.to(DEV), to(cache), table.to(DEV), n32), got)


def test_offsets_beyond_32_bits(hip_ext):
    """A cache of more than 2^32 elements: its last pages written, read and attended to."""
    print("[case] offsets", flush=True)
    g = gen(18)
    kv_heads, page_size, dim = 64, 256, 256
    pages = (1 << 32) // (kv_heads * page_size * dim) + 40
    cache = hip_ext.new_kv_cache(pages, kv_heads, page_size, dim, fp8=True, device=DEV)
    assert cache.key.numel() > 1 << 32
    n = 600
    table = torch.tensor([[pages - 1, pages - 3, pages - 2]], dtype=torch.int32, device=DEV)
    rows = [normal(g, 1, kv_heads, n, dim).to(torch.bfloat16) for _ in range(2)]
    starts, n32 = torch.zeros(1, dtype=torch.int32, device=DEV), torch.full((1,), n, dtype=torch.int32, device=DEV)
    hip_ext.kv_append(cache, *(r.to(DEV) for r in rows), table, starts)
    small = KVCache(*(t[pages - 3:].cpu() for t in cache))
    at = table.cpu() - (pages - 3)
    for data, scales, r in ((small.key, small.key_scales, rows[0]), (small.value, small.value_scales, rows[1])):
        p = torch.arange(n)
        page, slot = at[0, p // page_size].long(), p % page_size
        ref.check_codes(bits(data)[page, :, slot].view(F8), scales[page, :, slot], r[0].transpose(0, 1).double())
    assert bits(cache.key)[:pages - 3].max() == 0
    back = hip_ext.kv_read(cache, table, n32, n)[0]
    want, _ = ref.position_rows(small.key, small.key_scales, at[0], torch.arange(n))
    assert ((back[0].double().cpu() - want.transpose(0, 1)).abs() <= (ref.BF16 * (1 + ref.U) + ref.U) * want.transpose(0, 1).abs()).all()
    q = normal(g, 1, kv_heads, dim).to(torch.bfloat16)
    got = hip_ext.paged_attention(q.to(DEV), cache, table, n32)
    ref.check_attention(got, q, small, at, n32, dim ** -0.5)


# ---------------------------------------------------------- used together --
@pytest.mark.parametrize("fp8", [False, True])
def test_decode_steps_together(hip_ext, fp8):
    """A prompt appended, then tokens one by one, each attended to: eager, and
    replayed from a captured graph whose counters advance on the device."""
    print(f"[case] decode together {fp8}", flush=True)
    g = gen(19)
    batch, heads, kv_heads, page_size, dim, steps = 3, 8, 4, 16, 64, 40
    prompt = [0, 30, 301]
    table, pages = make_table(g, [n + steps for n in prompt], page_size)
    cache = hip_ext.new_kv_cache(pages, kv_heads, page_size, dim, fp8=fp8, device=DEV)
    held = hip_ext.new_kv_cache(pages, kv_heads, page_size, dim, fp8=fp8, device=DEV)
    dtable = table.to(DEV)
    rows = [normal(g, batch, kv_heads, 301, dim).to(torch.bfloat16).to(DEV) for _ in range(2)]
    counts = torch.tensor(prompt, dtype=torch.int32, device=DEV)
    new = [normal(g, steps, batch, kv_heads, 1, dim).to(torch.bfloat16).to(DEV) for _ in range(2)]
    queries = normal(g, steps, batch, heads, dim).to(torch.bfloat16).to(DEV)
    zeros = torch.zeros_like(counts)
    for c in (cache, held):
        hip_ext.kv_append(c, *rows, dtable, zeros, counts)
    want = []
    for i in range(steps):
        hip_ext.kv_append(cache, new[0][i], new[1][i], dtable, counts + i)
        want.append(hip_ext.paged_attention(queries[i], cache, dtable, counts + i + 1))
        if i % 13 == 0:
            ref.check_attention(want[-1], queries[i], cache, table, counts + i + 1, dim ** -0.5)
    key, query, value = new[0][0].clone(), queries[0].clone(), new[1][0].clone()
    starts, lengths = counts.clone(), counts + 1
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        hip_ext.kv_append(held, key, value, dtable, starts)
        out = hip_ext.paged_attention(query, held, dtable, lengths)
        starts.add_(1)
        lengths.add_(1)
    for i in range(steps):
        key.copy_(new[0][i])
        value.copy_(new[1][i])
        query.copy_(queries[i])
        graph.replay()
        hip_ext.paged_attention(queries[0], cache, dtable, counts)  # eager work between the replays
        torch.cuda.synchronize()
        assert torch.equal(out, want[i]), f"step {i}"
    for a, b in zip(cache, held):
        assert a is None or torch.equal(bits(a), bits(b))


@pytest.mark.parametrize("fp8", [False, True])
def test_a_captured_call_follows_lengths_and_pages(hip_ext, fp8):
    """One graph, replayed with other lengths, tables and queries in its buffers: other
    sequences are short, long and empty each time, and lie in other columns."""
    print(f"[case] captured lengths {fp8}", flush=True)
    g = gen(22)
    most = [9000, 700, 4000, 130, 2500]
    cache, table = filled(g, most, 2, 32, 64, fp8)
    kv = to(cache)
    dtable, n32, q = table.to(DEV), torch.zeros(5, dtype=torch.int32, device=DEV), torch.zeros(5, 6, 64, dtype=torch.bfloat16, device=DEV)
    hip_ext.paged_attention(q, kv, dtable, n32)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = hip_ext.paged_attention(q, kv, dtable, n32)
    for share in ([1, 1, 1, 1, 1], [0, 0, 1, 0.5, 0], [0.01, 1, 0, 0, 0.9], [0, 0, 0, 0, 0], [0.5, 0.3, 0.2, 1, 0.1], [1, 0, 0, 0, 0]):
        lengths = torch.tensor([int(n * f) for n, f in zip(most, share)], dtype=torch.int32)
        query = normal(g, 5, 6, 64).to(torch.bfloat16)
        n32.copy_(lengths)
        q.copy_(query)
        graph.replay()
        want = hip_ext.paged_attention(q, kv, dtable, n32)  # eager work between the replays
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        ref.check_attention(out, query, cache, table, lengths, 0.125)


def test_every_code_is_its_value(hip_ext):
    """Each of the 256 codes as a value, attended to alone, and read back: exact (both NaN codes NaN)."""
    print("[case] codes", flush=True)
    codes = torch.arange(256, dtype=torch.int32).to(torch.uint8)
    cache = hip_ext.new_kv_cache(1, 1, 16, 256, fp8=True, device=DEV)
    bits(cache.value)[0, 0, 0] = codes.to(DEV)
    cache.value_scales[0, 0, 0] = 0.5
    one = torch.ones(1, dtype=torch.int32, device=DEV)
    out = hip_ext.paged_attention(torch.ones(1, 2, 256, dtype=torch.bfloat16, device=DEV), cache, one.view(1, 1) - 1, one)
    read = hip_ext.kv_read(cache, one.view(1, 1) - 1, one, 1)[1]
    want = codes.view(F8).float() * 0.5
    assert want.isnan().sum() == 2
    for got in (out[0, 0], out[0, 1], read[0, 0, 0]):
        assert torch.equal(got.float().cpu().nan_to_num(1e9), want.nan_to_num(1e9))


def test_another_stream_than_the_tensors(hip_ext):
    """Written on one stream, attended to on another one behind it."""
    print("[case] other stream", flush=True)
    g = gen(23)
    rows = [normal(g, 2, 4, 900, 64).to(torch.bfloat16).to(DEV) for _ in range(2)]
    q = normal(g, 2, 8, 64).to(torch.bfloat16).to(DEV)
    cache = hip_ext.new_kv_cache(60, 4, 32, 64, fp8=True, device=DEV)
    table = torch.randperm(60, generator=g)[:58].view(2, 29).to(torch.int32).to(DEV)
    starts, n32 = torch.zeros(2, dtype=torch.int32, device=DEV), torch.tensor([900, 41], dtype=torch.int32, device=DEV)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    with torch.cuda.stream(streams[0]):
        hip_ext.kv_append(cache, *rows, table, starts, n32)
    streams[1].wait_stream(streams[0])
    with torch.cuda.stream(streams[1]):
        out = hip_ext.paged_attention(q, cache, table, n32)
    torch.cuda.synchronize()
    ref.check_attention(out, q, to(cache, "cpu"), table, n32, 0.125)


def test_calls_on_two_streams_at_once(hip_ext):
    print("[case] two streams", flush=True)
    g = gen(20)
    cache, table = filled(g, [9000, 4000], 4, 16, 128, True)
    kv, dtable = to(cache), table.to(DEV)
    n32 = torch.tensor([9000, 4000], dtype=torch.int32, device=DEV)
    q = normal(g, 2, 2, 8, 128).to(torch.bfloat16).to(DEV)
    want = [hip_ext.paged_attention(x, kv, dtable, n32) for x in q]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(hip_ext.paged_attention(q[i], kv, dtable, n32))
    torch.cuda.synchronize()
    assert all(torch.equal(t, want[i]) for i in range(2) for t in got[i])


def test_two_graphs_at_once(hip_ext):
    """Two captured graphs replayed on two streams: neither's workspace is the other's."""
    print("[case] two graphs", flush=True)
    g = gen(21)
    cache, table = filled(g, [9000, 4000], 4, 16, 128, False)
    kv, dtable = to(cache), table.to(DEV)
    n32 = torch.tensor([9000, 4000], dtype=torch.int32, device=DEV)
    q = normal(g, 2, 2, 8, 128).to(torch.bfloat16).to(DEV)
    want = [hip_ext.paged_attention(x, kv, dtable, n32) for x in q]
    streams, graphs, outs = [torch.cuda.Stream() for _ in range(2)], [], []
    torch.cuda.synchronize()
    for x, s in zip(q, streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            outs.append(hip_ext.paged_attention(x, kv, dtable, n32))
        graphs.append(graph)
    for _ in range(20):
        for o in outs:
            o.fill_(7)
        torch.cuda.synchronize()
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
