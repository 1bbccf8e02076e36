"""The paged key-value cache and its attention in 64 bits, and how far the kernels
may be from them. Tolerances are derived, not measured; U = 2^-24 is half a step of
FP32, a BF16 rounding is off by at most 2^-8 of the value."""

from __future__ import annotations

import torch

U = 2.0 ** -24
BF16 = 2.0 ** -8
FP8_MAX = 448.0


def quantize(v):
    """Codes and scales of v [..., dim] for a cache that the tests fill themselves."""
    most = v.abs().amax(-1)
    d = torch.where(most == 0, torch.ones_like(most), (most / FP8_MAX).clamp_min(2.0 ** -126))
    return (v / d[..., None]).to(torch.float8_e4m3fn), d


def take(pages, index):
    """pages[index], also of 8-bit floats."""
    if pages.dtype is torch.float8_e4m3fn:
        return pages.view(torch.uint8)[index].view(torch.float8_e4m3fn)
    return pages[index]


def position_rows(pages, scales, table_row, positions):
    """Values [positions, kv_heads, dim] in float64 of one sequence (CPU tensors) and
    which of the positions have a page."""
    page_size = pages.shape[2]
    entry, slot = positions // page_size, positions % page_size
    inside = entry < table_row.numel()
    page = torch.full_like(positions, -1)
    page[inside] = table_row[entry[inside]].long()
    there = (page >= 0) & (page < pages.shape[0])
    at = page.clamp(0, pages.shape[0] - 1)
    rows = take(pages, (at, slice(None), slot)).double()
    if scales is not None:
        rows = rows * scales[at, :, slot].double()[..., None]
    return rows, there


def attention64(query, cache, table, lengths, scale, window=None):
    """(output [batch, heads, dim], tolerance) in float64 on the CPU.

    The score of a position is an FP32 sum of dim exact products: 2 U each (the
    matrix cores may cut) of the sum of magnitudes, then the scales' products (3 U)
    and the base's change, so off by e = scale * (2 dim + 8) U sum|q k| + 4 U |s|.
    Its weight exp(s - m) is off by the factor e + 4 U (|s| + |m|) + 4 U, and by
    4 U each time that the running maximum moves, at most once per 16 positions.
    Sums of n weights and of n weighted values add 2 n U of their magnitudes. A
    weight is multiplied with values as two BF16 numbers: 2^-16 of it is lost. The
    joins of partial results (at most 1024) add as many 4 U. Last the division and
    one BF16 rounding."""
    query, table, lengths = query.double().cpu(), table.cpu(), lengths.cpu()
    key, value, ks, vs = (None if t is None else t.cpu() for t in cache)
    batch, heads, dim = query.shape
    group = heads // key.shape[1]
    out, tol = torch.zeros_like(query), torch.zeros_like(query)
    capacity = table.shape[1] * key.shape[2]
    for b in range(batch):
        n = min(max(int(lengths[b]), 0), capacity)
        positions = torch.arange(max(0, n - window) if window else 0, n)
        k, there = position_rows(key, ks, table[b], positions)
        v, _ = position_rows(value, vs, table[b], positions)
        k, v = k[there], v[there]
        n = k.shape[0]
        if n == 0:
            continue
        k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)  # [n, heads, dim]
        products = k * query[b]
        s = scale * products.sum(2)
        w = torch.softmax(s, 0)
        out[b] = (w[..., None] * v).sum(0)
        most = s.abs().amax(0)
        e = abs(scale) * (2 * dim + 8) * U * products.abs().sum(2) + 4 * U * s.abs()
        off = e.amax(0) + 8 * U * most + 4 * U + 4 * U * (n // 16 + 1 + 1024)
        off = 2 * off + 2.0 ** -16 + 4 * n * U + 8 * U  # (weights above and below the fraction's line)
        tol[b] = (w[..., None] * v.abs()).sum(0) * off[:, None]
    return out, tol * (1 + BF16) + BF16 * out.abs() + 2.0 ** -133


def check_attention(got, query, cache, table, lengths, scale, window=None):
    want, tol = attention64(query, cache, table, lengths, scale, window)
    off = (got.double().cpu() - want).abs() - tol
    assert torch.isfinite(got).all(), "not finite"
    assert (off <= 0).all(), f"{int((off > 0).sum())} of {off.numel()} outside, worst by {float(off.max()):.3e}"


def check_codes(codes, scales, rows):
    """Codes [..., dim] and scales of ``rows`` (float64, finite): a code is e4m3(v')
    with v' = v / d but for three FP32 roundings (scale, reciprocal, product), so
    within 2^-4 of v / d (or half a subnormal step, 2^-10)."""
    most = rows.abs().amax(-1)
    d = torch.where(most == 0, torch.ones_like(most), (most / FP8_MAX).clamp_min(2.0 ** -126))
    codes, scales = codes.double().cpu(), scales.double().cpu()
    assert ((scales - d).abs() <= 2 * U * d).all(), "scales"
    v = rows / d[..., None]
    slack = torch.maximum(2.0 ** -4 * v.abs() * (1 + 3 * U), torch.full_like(v, 2.0 ** -10)) + 3 * U * v.abs()
    assert ((codes - v).abs() <= slack).all(), "codes"
