"""The 8-bit operators on the GPU against their definition in 64 bits (tolerances
in fp8_reference.py), at the sizes and values where they can go wrong."""

from __future__ import annotations

import pytest
import torch

import fp8_cases
import fp8_reference as ref
from uma_qmoe_amd.native_backend import Fp8Matrix

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def note(msg):
    print(f"[case] {msg}", flush=True)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def normal(g, *shape, std=1.0):
    return (std * torch.randn(*shape, generator=g)).to(torch.bfloat16)


def on_gpu(t, offset=0):
    """A device copy whose first element lies ``offset`` elements behind an
    allocation's start (not 16-byte aligned for odd offsets)."""
    flat = torch.empty(t.numel() + offset, dtype=t.dtype, device=DEV)
    flat[offset:] = t.to(DEV).reshape(-1)
    return flat[offset:].view(t.shape)


# ------------------------------------------------------------- row operators --
# one group, its ends, several; the 1-, 2- and 4-pass rows and longer ones; not multiples of 8
COLS = [1, 7, 8, 120, 127, 128, 129, 136, 511, 512, 520, 1400, 2047, 2048, 2056, 4104, 5632, 8192, 8200, 8201, 20000]


@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("rows,offset", [(1, 0), (5, 0), (3, 1), (37, 3)])
@pytest.mark.parametrize("residual", [False, True])
def test_add_rmsnorm(hip_ext, rows, cols, offset, residual):
    note(f"add_rmsnorm {rows}x{cols}+{offset} residual={residual}")
    g = gen(cols + rows)
    x, r = normal(g, rows, cols), normal(g, rows, cols, std=4.0) if residual else None
    w = (1 + 0.1 * torch.randn(cols, generator=g)).to(torch.bfloat16) if rows != 5 else None
    s = x if r is None else (x.float() + r.float()).to(torch.bfloat16)
    y = ref.rmsnorm64(s.double(), 1e-6, None if w is None else w.double())
    delta = ref.rmsnorm_delta(cols)
    xd, rd, wd = on_gpu(x, offset), None if r is None else on_gpu(r, offset), None if w is None else on_gpu(w, offset)
    total, n, q = hip_ext.add_rmsnorm(xd, rd, 1e-6, wd, bf16=True, fp8=True)
    if r is None:
        assert total is xd
    else:
        assert torch.equal(total.cpu(), s)
        assert torch.equal(xd.cpu(), x) and torch.equal(rd.cpu(), r)
    # two BF16 roundings (the norm, its product with the weight)
    assert ((n.double().cpu() - y).abs() <= ((1 + ref.BF16) ** 2 * (1 + delta) - 1) * y.abs()).all()
    ref.check_fp8(q.codes, q.scales, y, 1, delta)
    # one output alone gives the same bits, and so does the sum in the residual's place
    only = hip_ext.add_rmsnorm(xd, rd, 1e-6, wd, bf16=True, fp8=False)
    assert only[2] is None and torch.equal(only[1], n)
    keep = None if rd is None else rd.clone()
    only = hip_ext.add_rmsnorm(xd, keep, 1e-6, wd, bf16=False, fp8=True, inplace=keep is not None)
    assert only[1] is None and torch.equal(only[2].codes.view(torch.uint8), q.codes.view(torch.uint8))
    assert torch.equal(only[2].scales, q.scales)
    if keep is not None:
        assert only[0] is keep and torch.equal(keep, total)


@pytest.mark.parametrize("rows,cols", [(9, 120), (5, 512), (64, 2048), (7, 8200), (3, 1401)])
def test_add_rmsnorm_rounds_its_norm_once(hip_ext, rows, cols):
    """The BF16 output is the FP32 value of w * n, whose codes the 8-bit output
    holds, rounded once."""
    note(f"add_rmsnorm rounds once {rows}x{cols}")
    g = gen(rows)
    x, r = normal(g, rows, cols), normal(g, rows, cols, std=4.0)
    w = (1 + 0.3 * torch.randn(cols, generator=g)).to(torch.bfloat16)
    total, n, _ = hip_ext.add_rmsnorm(x.to(DEV), r.to(DEV), 1e-6, w.to(DEV), fp8=True)
    y = ref.rmsnorm64(total.double().cpu(), 1e-6, w.double())
    assert ((n.double().cpu() - y).abs() <= ((1 + ref.BF16) * (1 + ref.rmsnorm_delta(cols)) - 1) * y.abs()).all()


@pytest.mark.parametrize("rows,cols", [(1, 2048), (5, 100), (4, 400), (3, 2047), (2, 8201), (2, 20000)])
def test_add_rmsnorm_sum_in_an_input(hip_ext, rows, cols):
    """The sum over the input, over the residual, and over one tensor that is both:
    the same bits as into a tensor of its own."""
    note(f"add_rmsnorm sum in an input {rows}x{cols}")
    g = gen(cols)
    x, r = normal(g, rows, cols).to(DEV), normal(g, rows, cols).to(DEV)
    w = (1 + 0.1 * torch.randn(cols, generator=g)).to(torch.bfloat16).to(DEV)
    stream = torch.cuda.current_stream().cuda_stream

    def into(a, b, total):
        out, codes = torch.empty_like(a), torch.empty(rows, cols, dtype=torch.uint8, device=DEV)
        scales = torch.empty(rows, -(-cols // 128), device=DEV)
        assert hip_ext.lib.uqm_add_rmsnorm(a.data_ptr(), b.data_ptr(), rows, cols, w.data_ptr(), 1e-6, total.data_ptr(),
                                           out.data_ptr(), codes.data_ptr(), scales.data_ptr(), stream) == 0
        return total, out, codes, scales

    def same(got, want):
        return all(torch.equal(a, b) for a, b in zip(got, want))

    want = into(x, r, torch.empty_like(x))
    over_x, over_r = x.clone(), r.clone()
    assert same(into(over_x, r, over_x), want) and same(into(x, over_r, over_r), want)
    twice, both = into(x, x, torch.empty_like(x)), x.clone()
    assert same(into(both, both, both), twice)


def test_add_rmsnorm_rounds_as_rmsnorm(hip_ext):
    """The BF16 output is uqm_rmsnorm's of the same sum: both divide by the same
    root up to the order of its sum, so at most one step of each rounding."""
    note("add_rmsnorm against rmsnorm")
    g = gen(3)
    for rows, cols in ((7, 2048), (3, 8192), (4, 100)):
        x, r, w = normal(g, rows, cols).to(DEV), normal(g, rows, cols).to(DEV), normal(g, cols).to(DEV)
        total, n, _ = hip_ext.add_rmsnorm(x, r, 1e-6, w)
        want = hip_ext.rmsnorm(total, 1e-6, w).float()
        assert ((n.float() - want).abs() <= 2 * 2.0 ** -7 * want.abs()).all()


@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("rows,offset", [(1, 0), (37, 0), (3, 1)])
def test_silu_mul(hip_ext, rows, cols, offset):
    note(f"silu_mul {rows}x{cols}+{offset}")
    x = normal(gen(cols + rows), rows, 2 * cols, std=4.0)
    g, u = x[:, :cols].double(), x[:, cols:].double()
    y, delta = ref.silu64(g, u), ref.silu_delta(g)
    xd = on_gpu(x, offset)
    out, q = hip_ext.silu_mul(xd, bf16=True, fp8=True)
    assert ((out.double().cpu() - y).abs() <= ((1 + ref.BF16) * (1 + delta) - 1) * y.abs() + 2.0 ** -133).all()
    ref.check_fp8(q.codes, q.scales, y, 1, delta)
    assert torch.equal(hip_ext.silu_mul(xd)[0], out)
    only = hip_ext.silu_mul(xd, bf16=False, fp8=True)
    assert only[0] is None and torch.equal(only[1].codes.view(torch.uint8), q.codes.view(torch.uint8))


def test_silu_mul_at_the_ends(hip_ext):
    """Gates whose exponential overflows, infinities and NaN."""
    note("silu_mul ends")
    inf, nan = float("inf"), float("nan")
    g = torch.tensor([-88.0, -89.0, -100.0, -3e38, 88.0, 100.0, 3e38, inf, -inf, nan, 0.0, -0.0], dtype=torch.bfloat16)
    x = torch.zeros(1, 256, dtype=torch.bfloat16)
    x[0, :len(g)] = g
    x[0, 128:] = 1.0
    out, q = hip_ext.silu_mul(x.to(DEV), bf16=True, fp8=True)
    got = out.float().cpu()[0]
    assert (got[:4].abs() <= 1e-35).all()  # 88 exp(-88) is 5e-37
    assert torch.equal(got[4:8], g[4:8].float())
    assert got[8].isnan() and got[9].isnan() and (got[10:] == 0).all()
    assert q.scales.isnan().all() and q.codes.float().isnan().all()


@pytest.mark.parametrize("cols", [16, 48, 130, 384, 648])
def test_silu_mul_rows_keep_to_themselves(hip_ext, cols):
    """A wave holds several narrow rows, or parts of two: gates whose exponential
    overflows, infinities and NaN in every third row change no bit of the others."""
    note(f"silu_mul rows {cols}")
    x = normal(gen(cols), 3000, 2 * cols, std=4.0)
    ends = x.clone()
    ends[::3, :7] = torch.tensor([-88.0, -100.0, -3e38, float("-inf"), float("inf"), float("nan"), 3e38], dtype=torch.bfloat16)
    want, q = hip_ext.silu_mul(x.to(DEV), fp8=True)
    got, p = hip_ext.silu_mul(ends.to(DEV), fp8=True)
    for rows in (slice(1, None, 3), slice(2, None, 3)):
        assert torch.equal(p.scales[rows], q.scales[rows])
        assert torch.equal(p.codes[rows].view(torch.uint8), q.codes[rows].view(torch.uint8))
        assert torch.equal(got[rows], want[rows])
    # and the other values of a row in BF16 neither
    assert torch.equal(got[::3, 7:], want[::3, 7:])


@pytest.mark.parametrize("block", [1, 128])
@pytest.mark.parametrize("rows,offset", [(1, 0), (127, 0), (128, 1), (129, 0), (300, 0)])
@pytest.mark.parametrize("cols", [1, 8, 120, 128, 129, 136, 1400, 2048, 2056])
def test_quantize_bits(hip_ext, rows, cols, offset, block):
    """The input is exact, so every rounding is known: scale, reciprocal,
    product, and the conversion torch makes on the CPU."""
    note(f"fp8_quantize {rows}x{cols}+{offset} block={block}")
    x = normal(gen(rows + cols), rows, cols) * torch.exp2(torch.randint(-20, 20, (rows, 1), generator=gen(rows)))
    x = x.to(torch.bfloat16)
    q = hip_ext.fp8_quantize(on_gpu(x, offset), block_rows=block)
    m = ref.block_max(x.float(), block)
    d = torch.where(m == 0, torch.ones_like(m), (m / 448.0).clamp_min(2.0 ** -126))
    assert torch.equal(q.scales.cpu(), d)
    want = (x.float() * ref.each(1.0 / d, block, rows, cols)).to(torch.float8_e4m3fn)
    # (element by element: -0 is 0)
    assert torch.equal(q.codes.cpu().float(), want.float())
    ref.check_fp8(q.codes, q.scales, x.double(), block, 0.0)


@pytest.mark.parametrize("block", [1, 128])
def test_quantize_takes_a_nearest_code(hip_ext, block):
    """No e4m3 value is nearer to v / d than the code, but by the roundings of 1 / d
    and of its product with v (U each). BF16 values are often the middle between
    two codes, up to them: 0.80859375 beside 1.078125 is 336, between 320 and 352."""
    note(f"fp8_quantize nearest block={block}")
    x = normal(gen(12), 256, 512)
    x[:128, :128] = x[:128, :128].clamp(-1, 1)
    x[:128, 0] = 1.078125
    x[:128, 1] = 0.80859375
    q = hip_ext.fp8_quantize(x.to(DEV), block_rows=block)
    v = x.double() / ref.each(q.scales.double().cpu(), block, *x.shape)
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    codes = codes[codes.isfinite()].sort().values
    at = torch.searchsorted(codes, v).clamp(1, len(codes) - 1)
    nearest = torch.minimum((v - codes[at - 1]).abs(), (v - codes[at]).abs())
    off = (q.codes.double().cpu() - v).abs()
    assert (off <= nearest + 2 * 2.001 * ref.U * v.abs()).all()
    assert q.codes[0, 1].item() in (320, 352)


@pytest.mark.parametrize("block", [1, 128])
def test_quantize_ends(hip_ext, block):
    """Groups of zeros, of the smallest and largest values, with a NaN or an
    infinity; every one beside an ordinary group that is left alone."""
    note(f"fp8_quantize ends block={block}")
    big = torch.finfo(torch.bfloat16).max
    rows = 128 * 6 if block == 128 else 6
    x = normal(gen(1), rows, 256)
    of = [x[i * block:(i + 1) * block, :128] for i in range(6)]
    of[0].zero_()
    of[1].fill_(2.0 ** -133)  # the smallest BF16 value
    of[2].fill_(-big)
    of[3][0, 5] = float("nan")
    of[4][0, 6] = float("-inf")
    of[5].fill_(-0.0)
    q = hip_ext.fp8_quantize(x.to(DEV), block_rows=block)
    s, c = q.scales.cpu(), q.codes.float().cpu()
    at = [c[i * block:(i + 1) * block, :128] for i in range(6)]
    assert s[0, 0] == 1 and (at[0] == 0).all() and s[5, 0] == 1 and (at[5] == 0).all()
    assert s[1, 0] == 2.0 ** -126 and (at[1] == 2.0 ** -7).all()
    assert s[2, 0] == torch.tensor(big) / 448 and (at[2] == -448).all()
    assert s[3, 0].isnan() and at[3].isnan().all()
    assert s[4, 0] == float("inf") and at[4][0, 6].isnan()
    at[4][0, 6] = 0
    assert (at[4] == 0).all()
    ref.check_fp8(c[:, 128:], s[:, 1:], x[:, 128:].double(), block, 0.0)


def test_quantize_with_scales_next_to_the_input(hip_ext):
    """Blocks of 128 rows have few scales: the ones of 4095 x 128 right before the
    input, or right behind the codes, overlap nothing."""
    note("fp8_quantize scales next to the input")
    rows, cols = 4095, 128
    groups = -(-rows // 128)
    room = torch.zeros(4 * 4096 + 2 * rows * cols, dtype=torch.uint8, device=DEV)
    scales = room[4 * 4096 - 4 * groups:4 * 4096].view(torch.float32)
    x = room[4 * 4096:].view(torch.bfloat16).view(rows, cols)
    x.copy_(normal(gen(2), rows, cols))
    codes = torch.empty(rows, cols, dtype=torch.uint8, device=DEV)
    stream = torch.cuda.current_stream().cuda_stream
    assert hip_ext.lib.uqm_fp8_quantize(x.data_ptr(), rows, cols, 128, codes.data_ptr(), scales.data_ptr(), stream) == 0
    want = hip_ext.fp8_quantize(x, block_rows=128)
    assert torch.equal(codes, want.codes.view(torch.uint8)) and torch.equal(scales, want.scales.flatten())


def test_norm_and_sum_keep_nan_and_infinity(hip_ext):
    """A row with a NaN or an infinity is lost (as in rmsnorm), its neighbours are not."""
    note("add_rmsnorm nan")
    g = gen(9)
    x, r = normal(g, 4, 300), normal(g, 4, 300)
    x[1, 7] = float("nan")
    r[2, 299] = float("inf")
    total, n, q = hip_ext.add_rmsnorm(x.to(DEV), r.to(DEV), fp8=True)
    assert total.isnan().sum() == 1 and total.isinf().sum() == 1
    for row in (1,):
        assert n[row].isnan().all() and q.scales[row].isnan().all()
    assert q.codes[2].float().isnan().any() and q.scales[2].isnan().any()
    for row in (0, 3):
        assert n[row].isfinite().all() and q.codes[row].float().isfinite().all()


def test_strided_and_batched_inputs(hip_ext):
    note("strided and batched row operators")
    g = gen(4)
    base = normal(g, 6, 3, 512).to(DEV)
    x = base[::2, :, 100:356]
    flat = x.reshape(-1, 256).contiguous()
    for fn in (lambda v: hip_ext.add_rmsnorm(v, v, fp8=True)[2], lambda v: hip_ext.silu_mul(v, fp8=True)[1],
               lambda v: hip_ext.fp8_quantize(v)):
        got, want = fn(x), fn(flat)
        assert got.codes.shape[:-1] == (3, 3) and got.scales.shape[:-1] == (3, 3)
        assert torch.equal(got.codes.view(torch.uint8).flatten(), want.codes.view(torch.uint8).flatten())
        assert torch.equal(got.scales.flatten(), want.scales.flatten())
    for rows in (0,):
        none = hip_ext.add_rmsnorm(base[:0, 0], base[:0, 1], fp8=True)
        assert none[1].shape == (0, 512) and none[2].scales.shape == (0, 4)
        assert hip_ext.silu_mul(base[:0, 0])[0].shape == (0, 256)
        assert hip_ext.fp8_quantize(base[:0, 0], block_rows=128).scales.shape == (0, 4)


# -------------------------------------------------------------------- product --
def operands(t, n, k, seed, bias=True):
    g = gen(seed)
    codes = (100 * torch.randn(t, k, generator=g)).clamp(-448, 448).to(torch.float8_e4m3fn)
    w = (100 * torch.randn(n, k, generator=g)).clamp(-448, 448).to(torch.float8_e4m3fn)
    blocks = -(-k // 128)
    scales = torch.exp2(8 * torch.rand(t, blocks, generator=g) - 10)
    ws = torch.exp2(8 * torch.rand(-(-n // 128), blocks, generator=g) - 16)
    b = normal(g, n, std=30.0) if bias else None
    return codes, scales, w, ws, b


def product(ext, codes, scales, w, ws, b):
    return ext.fp8_linear(Fp8Matrix(codes.to(DEV), scales.to(DEV)), Fp8Matrix(w.to(DEV), ws.to(DEV), 128),
                          None if b is None else b.to(DEV))


LINEAR = [(1, 1, 16), (1, 16, 128), (1, 17, 144), (2, 200, 112), (1, 384, 2048), (15, 129, 272), (16, 64, 128),
          (17, 15, 256), (31, 256, 1040), (33, 127, 384), (64, 300, 512), (65, 96, 640), (100, 1000, 2000),
          (127, 257, 528), (128, 256, 1024), (129, 130, 1152), (255, 513, 384), (256, 256, 256), (300, 640, 2048),
          (513, 384, 144), (777, 1410, 656), (1, 2048, 5632), (5, 11264, 256), (32, 2048, 2816),
          # tiles of the large-tile kernel: whole and ragged in each direction, one block of columns, a short last one
          (2048, 2048, 128), (2049, 2049, 384), (2100, 2300, 272), (4200, 1100, 1040), (1030, 4100, 16)]


@pytest.mark.parametrize("t,n,k", LINEAR)
@pytest.mark.parametrize("bias", [False, True])
def test_linear(hip_ext, t, n, k, bias):
    note(f"fp8_linear {t}x{n}x{k} bias={bias}")
    args = operands(t, n, k, t + n + k, bias)
    y, tol = ref.linear64(*args)
    got = product(hip_ext, *args)
    assert got.dtype == torch.bfloat16 and got.shape == (t, n)
    off = (got.double().cpu() - y).abs() - tol
    assert (off <= 0).all(), f"{int((off > 0).sum())} of {off.numel()} outside, worst by {float(off.max()):.3e}"
    assert torch.equal(product(hip_ext, *args), got)  # no order of sums that changes


@pytest.mark.parametrize("t,n,k", [(3, 40, 144), (40, 300, 272), (200, 300, 400), (600, 520, 272), (2100, 2100, 400)])
def test_linear_confines_nan(hip_ext, t, n, k):
    """A row of NaN codes or scales (a neighbour's last, short block reads up to
    it) changes its own results only."""
    note(f"fp8_linear nan {t}x{n}x{k}")
    codes, scales, w, ws, b = operands(t, n, k, 5)
    y, tol = ref.linear64(codes, scales, w, ws, b)
    bad_t, bad_s, bad_n = t // 2, t - 1, n // 3
    nan8 = torch.full((k,), 0x7F, dtype=torch.uint8).view(torch.float8_e4m3fn)
    codes[bad_t], w[bad_n] = nan8, nan8
    scales[bad_s] = float("inf")
    got = product(hip_ext, codes, scales, w, ws, b).double().cpu()
    assert got[bad_t].isnan().all() and got[:, bad_n].isnan().all() and not got[bad_s].isfinite().any()
    keep = torch.ones(t, n, dtype=torch.bool)
    keep[bad_t] = keep[bad_s] = False
    keep[:, bad_n] = False
    assert ((got - y).abs() <= tol)[keep].all()


@pytest.mark.parametrize("t,n,k", [(1, 33, 128), (20, 33, 128), (130, 250, 256), (300, 515, 256), (2050, 2050, 256)])
def test_linear_leaves_its_surroundings(hip_ext, t, n, k):
    """Nothing is written before or behind the output."""
    note(f"fp8_linear surroundings {t}x{n}x{k}")
    codes, scales, w, ws, _ = (None if v is None else v.to(DEV) for v in operands(t, n, k, 6, False))
    room = torch.full((t * n + 2048,), 7.0, dtype=torch.bfloat16, device=DEV)
    out = room[1024:1024 + t * n]
    stream = torch.cuda.current_stream().cuda_stream
    assert hip_ext.lib.uqm_fp8_linear(codes.data_ptr(), scales.data_ptr(), t, w.data_ptr(), ws.data_ptr(), n, k, None,
                                      out.data_ptr(), stream) == 0
    want = hip_ext.fp8_linear(Fp8Matrix(codes, scales), Fp8Matrix(w, ws, 128))
    assert torch.equal(out.view(t, n), want)
    assert (room[:1024] == 7).all() and (room[1024 + t * n:] == 7).all()
    # an output that is aligned to its elements only
    shifted = room[1025:1025 + t * n]
    assert hip_ext.lib.uqm_fp8_linear(codes.data_ptr(), scales.data_ptr(), t, w.data_ptr(), ws.data_ptr(), n, k, None,
                                      shifted.data_ptr(), stream) == 0
    assert torch.equal(shifted.view(t, n), want)


@pytest.mark.parametrize("kernel,t,n,k", fp8_cases.PLANNED + fp8_cases.ONE_ROW)
def test_linear_kernels(hip_ext, kernel, t, n, k):
    """Every kernel, at whole and at ragged sizes: the product, again with the
    same bits, with rows lost to NaN that the others must not see, and at an
    output that is aligned to its elements only, with nothing written around it."""
    note(f"fp8_linear kernel {kernel} {t}x{n}x{k}")
    assert fp8_cases.plan(t, n, k) == kernel
    codes, scales, w, ws, b = (v.to(DEV) for v in operands(t, n, k, t + n + k))
    x, weight = Fp8Matrix(codes, scales), Fp8Matrix(w, ws, 128)
    y, tol = ref.linear64(codes, scales, w, ws, b, device=DEV)
    got = hip_ext.fp8_linear(x, weight, b)
    assert ((got.double() - y).abs() <= tol).all()
    assert torch.equal(hip_ext.fp8_linear(x, weight, b), got)
    room = torch.full((t * n + 2048,), 7.0, dtype=torch.bfloat16, device=DEV)
    for at in (1024, 1025):
        room.fill_(7.0)
        out = room[at:at + t * n]
        assert hip_ext.lib.uqm_fp8_linear(codes.data_ptr(), scales.data_ptr(), t, w.data_ptr(), ws.data_ptr(), n, k,
                                          b.data_ptr(), out.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(out.view(t, n), got)
        assert (room[:at] == 7).all() and (room[at + t * n:] == 7).all()
    bad_t, bad_s, bad_n = t // 2, t - 1, n // 3
    codes.view(torch.uint8)[bad_t] = 0x7F
    w.view(torch.uint8)[bad_n] = 0x7F
    scales[bad_s] = float("inf")
    lost = hip_ext.fp8_linear(x, weight, b)
    assert lost[bad_t].isnan().all() and lost[:, bad_n].isnan().all() and not lost[bad_s].isfinite().any()
    keep = torch.ones(t, n, dtype=torch.bool, device=DEV)
    keep[bad_t] = keep[bad_s] = False
    keep[:, bad_n] = False
    assert torch.equal(lost[keep], got[keep])


def test_linear_of_bf16_and_batches(hip_ext):
    note("fp8_linear of BF16 input")
    g = gen(8)
    x = normal(g, 2, 5, 384).to(DEV)
    w = hip_ext.fp8_quantize(normal(g, 200, 384, std=0.02).to(DEV), block_rows=128)
    q = hip_ext.fp8_quantize(x)
    got = hip_ext.fp8_linear(x, w)
    assert got.shape == (2, 5, 200) and torch.equal(got, hip_ext.fp8_linear(q, w))
    assert torch.equal(hip_ext.fp8_linear(x.transpose(0, 1), w), got.transpose(0, 1))
    assert hip_ext.fp8_linear(x[:, :0], w).shape == (2, 0, 200)
    part = Fp8Matrix(q.codes[:, 1::2], q.scales[:, 1::2])
    assert torch.equal(hip_ext.fp8_linear(part, w), got[:, 1::2])
    exact = (q.dequantize().double().reshape(-1, 384) @ w.dequantize().double().t()).cpu().view(2, 5, 200)
    assert ((got.double().cpu() - exact).norm() <= 2.0 ** -8 * exact.norm() * 1.01)


# ------------------------------------------------------------------- together --
def ffn(ext, hidden, residual, norm, gate_up, down):
    """The dense gated layer that the operators make together."""
    total, _, q = ext.add_rmsnorm(hidden, residual, 1e-6, norm, bf16=False, fp8=True)
    _, h = ext.silu_mul(ext.fp8_linear(q, gate_up), bf16=False, fp8=True)
    return total, ext.fp8_linear(h, down)


def ffn_inputs(ext, rows, hidden, inter, seed):
    g = gen(seed)
    x, r = normal(g, rows, hidden).to(DEV), normal(g, rows, hidden, std=2.0).to(DEV)
    norm = (1 + 0.1 * torch.randn(hidden, generator=g)).to(torch.bfloat16).to(DEV)
    gate_up = normal(g, 2 * inter, hidden, std=0.02).to(DEV)
    down = normal(g, hidden, inter, std=0.02).to(DEV)
    return x, r, norm, gate_up, down


@pytest.mark.parametrize("rows,hidden,inter", [(1, 256, 512), (6, 2048, 1408), (77, 400, 208), (300, 2048, 5632)])
def test_dense_layer(hip_ext, rows, hidden, inter):
    """Against the same layer in 64 bits on the unquantised weights: an e4m3
    value is off by at most 2^-4 of itself, 2^-4 / sqrt(3) in the mean square over
    a step. Three quantised factors enter an output linearly through gate or up
    (weight, norm) and twice again (down weight, activation); independent errors
    add in the mean square: sqrt(2 * 2 + 2) * 2^-4 / sqrt(3) = 0.09, and SiLU's
    slope reaches 1.1: 0.1 of the norm."""
    note(f"dense layer {rows}x{hidden}x{inter}")
    x, r, norm, gate_up, down = ffn_inputs(hip_ext, rows, hidden, inter, rows)
    total, y = ffn(hip_ext, x, r, norm, hip_ext.fp8_quantize(gate_up, block_rows=128),
                   hip_ext.fp8_quantize(down, block_rows=128))
    s = (x.float() + r.float()).to(torch.bfloat16)
    assert torch.equal(total, s)
    n = ref.rmsnorm64(s.double().cpu(), 1e-6, norm.double().cpu())
    gu = n @ gate_up.double().cpu().t()
    want = ref.silu64(gu[:, :inter], gu[:, inter:]) @ down.double().cpu().t()
    assert (y.double().cpu() - want).norm() <= 0.1 * want.norm()


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_dense_layer_in_a_graph_and_on_streams(hip_ext, rows):
    """Captured once and replayed on new inputs, with eager work between the
    replays, and run on two side streams at once: the eager results' bits."""
    note(f"dense layer graph {rows}")
    x, r, norm, gate_up, down = ffn_inputs(hip_ext, rows, 512, 384, 11)
    gate_up, down = hip_ext.fp8_quantize(gate_up, block_rows=128), hip_ext.fp8_quantize(down, block_rows=128)
    inputs = [(normal(gen(i), rows, 512).to(DEV), normal(gen(50 + i), rows, 512).to(DEV)) for i in range(4)]
    want = [ffn(hip_ext, a, b, norm, gate_up, down) for a, b in inputs]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ffn(hip_ext, x, r, norm, gate_up, down)
    for (a, b), (total, y) in zip(inputs, want):
        x.copy_(a)
        r.copy_(b)
        graph.replay()
        ffn(hip_ext, b, a, norm, gate_up, down)
        torch.cuda.synchronize()
        assert torch.equal(out[0], total) and torch.equal(out[1], y)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for i, (a, b) in enumerate(inputs):
        s = streams[i % 2]
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(ffn(hip_ext, a, b, norm, gate_up, down))
    for s in streams:
        s.synchronize()
    for (total, y), (total_w, y_w) in zip(got, want):
        assert torch.equal(total, total_w) and torch.equal(y, y_w)


# ------------------------------------------------------- offsets past 32 bits --
def repeated(rows, cols, seed):
    """[rows, cols] BF16 on the device whose rows differ, made from 127 of them."""
    base = normal(gen(seed), 127, cols).to(DEV)
    return base.repeat(-(-rows // 127), 1)[:rows]


def test_rows_past_32_bits(hip_ext):
    """4.6 GB of BF16: the last rows are those of a small call."""
    note("row operators past 32 bits")
    rows, cols = 70001, 32768
    x = repeated(rows, cols, 1)
    last = x[-130:].clone()
    for fn in (lambda v: hip_ext.add_rmsnorm(v, None, bf16=False, fp8=True)[2], lambda v: hip_ext.silu_mul(v, bf16=False, fp8=True)[1],
               lambda v: hip_ext.fp8_quantize(v)):
        big, small = fn(x), fn(last)
        assert torch.equal(big.codes[-130:].view(torch.uint8), small.codes.view(torch.uint8))
        assert torch.equal(big.scales[-130:], small.scales)
        del big
    big = hip_ext.fp8_quantize(x, block_rows=128)
    small = hip_ext.fp8_quantize(x[70001 // 128 * 128:], block_rows=128)
    assert torch.equal(big.codes[70001 // 128 * 128:].view(torch.uint8), small.codes.view(torch.uint8))
    assert torch.equal(big.scales[-1:], small.scales)
    del big
    total, n, _ = hip_ext.add_rmsnorm(x, x)
    want = hip_ext.add_rmsnorm(last, last)
    assert torch.equal(total[-130:], want[0]) and torch.equal(n[-130:], want[1])


@pytest.mark.parametrize("t,n,k", [(3, 140001, 32768), (140001, 17, 32768), (70001, 32776, 16), (300, 16777, 262144)])
def test_linear_past_32_bits(hip_ext, t, n, k):
    """Weight, activations or output of over 4 GB; the last results in 64 bits."""
    note(f"fp8_linear past 32 bits {t}x{n}x{k}")
    x = hip_ext.fp8_quantize(repeated(t, k, 2))
    w = hip_ext.fp8_quantize(repeated(n, k, 3), block_rows=128)
    got = hip_ext.fp8_linear(x, w)[-40:, -200:]
    n0 = n // 128 * 128 if n % 128 >= 100 or n < 256 else (n // 128 - 1) * 128  # a block border before the last 200 rows
    n0 = max(0, n0 - 128)
    y, tol = ref.linear64(x.codes[-40:], x.scales[-40:], w.codes[n0:], w.scales[n0 // 128:], None)
    y, tol = y[:, -200:], tol[:, -200:]
    assert ((got.double().cpu() - y).abs() <= tol).all()


@pytest.mark.parametrize("op,cols", [("norm", 513), ("quantize", 1025), ("silu", 1025)])
def test_more_rows_than_a_launch_has_room_for(hip_ext, op, cols):
    """2^24 workgroups of a row each are 2^32 threads."""
    note(f"{op} of more rows than a launch has room for")
    fn = {"norm": lambda v: hip_ext.add_rmsnorm(v, None, bf16=False, fp8=True)[2],
          "quantize": hip_ext.fp8_quantize,
          "silu": lambda v: hip_ext.silu_mul(v, bf16=False, fp8=True)[1]}[op]
    part = normal(gen(4), 4099, cols * (2 if op == "silu" else 1)).to(DEV)
    repeats = ((1 << 24) + 4098) // 4099 + 1
    x = part.repeat(repeats, 1)
    big, small = fn(x), fn(part)
    del x
    for i in (0, repeats // 2, repeats - 2, repeats - 1):  # the last two hold the second launch's rows
        rows = slice(4099 * i, 4099 * (i + 1))
        assert torch.equal(big.codes[rows].view(torch.uint8), small.codes.view(torch.uint8))
        assert torch.equal(big.scales[rows], small.scales)


def test_more_blocks_than_a_launch_has_room_for(hip_ext):
    """2^24 blocks; the last, in a launch of its own, has 127 rows."""
    note("blocks of more rows than a launch has room for")
    rows = (1 << 31) - 1
    part = normal(gen(5), 1024, 1).to(DEV)
    x = part.repeat(1 << 21, 1)[:rows]
    big, small = hip_ext.fp8_quantize(x, block_rows=128), hip_ext.fp8_quantize(part, block_rows=128)
    last = hip_ext.fp8_quantize(part[-128:-1], block_rows=128)
    del x
    assert big.scales.shape == (1 << 24, 1)
    for first in (0, rows // 2048 * 1024, rows - 2047):
        assert torch.equal(big.codes[first:first + 1024].view(torch.uint8), small.codes.view(torch.uint8))
        assert torch.equal(big.scales[first // 128:first // 128 + 8], small.scales)
    assert torch.equal(big.codes[-127:].view(torch.uint8), last.codes.view(torch.uint8))
    assert torch.equal(big.scales[-1:], last.scales)
