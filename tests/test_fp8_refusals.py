"""What the 8-bit operators refuse, without a GPU: the library's entry points
check their arguments before they look at the device, the wrappers before they
call the library."""

from __future__ import annotations

import ctypes

import pytest
import torch

import fp8_cases
from uma_qmoe_amd import _native
from uma_qmoe_amd.native_backend import Fp8Matrix, HipExtension

A, B, C, D, E = (1 << 20, 2 << 20, 3 << 20, 4 << 20, 5 << 20)  # addresses that nothing reads


@pytest.fixture(scope="module")
def lib():
    return _native.library()


def refused(lib, name, args, words):
    rc = getattr(lib, name)(*args, None)
    message = lib.uqm_last_error().decode()
    assert rc == 1, (rc, message)  # UQM_ERR_ARGUMENT
    assert words in message, message


@pytest.mark.parametrize("args,words", [
    ((A, None, -1, 128, None, 1e-6, None, B, None, None), "rows"),
    ((A, None, 1 << 31, 128, None, 1e-6, None, B, None, None), "rows"),
    ((A, None, 4, 0, None, 1e-6, None, B, None, None), "columns"),
    ((A, None, 4, 128, None, -1e-6, None, B, None, None), "eps"),
    ((A, None, 4, 128, None, float("nan"), None, B, None, None), "eps"),
    ((A, C, 4, 128, None, 1e-6, None, B, None, None), "residual and sum"),
    ((A, None, 4, 128, None, 1e-6, C, B, None, None), "residual and sum"),
    ((A, None, 4, 128, None, 1e-6, None, None, None, None), "no output"),
    ((A, None, 4, 128, None, 1e-6, None, B, D, None), "together"),
    ((A, None, 4, 128, None, 1e-6, None, B, None, D), "together"),
    ((None, None, 4, 128, None, 1e-6, None, B, None, None), "required"),
    ((A + 1, None, 4, 128, None, 1e-6, None, B, None, None), "aligned"),
    ((A, None, 4, 128, None, 1e-6, None, B, D, E + 2), "aligned"),
    ((A, None, 4, 128, None, 1e-6, None, A, None, None), "overlaps an input"),
    ((A, B, 4, 128, None, 1e-6, A + 2, C, None, None), "overlaps an input"),
    ((A, B, 4, 128, C, 1e-6, B, C + 254, None, None), "overlaps an input"),
    ((A, B, 4, 128, None, 1e-6, C, C + 1022, None, None), "outputs overlap"),
    ((A, None, 4, 128, None, 1e-6, None, B, B + 1020, D), "outputs overlap"),
])
def test_add_rmsnorm(lib, args, words):
    refused(lib, "uqm_add_rmsnorm", args, words)


@pytest.mark.parametrize("rows", [1, 4])
def test_add_rmsnorm_keeps_its_weight(lib, rows):
    """The sum may be written over the input or the residual, never over the
    weight, which of one row has as many bytes."""
    refused(lib, "uqm_add_rmsnorm", (A, B, rows, 128, C, 1e-6, C, D, None, None), "overlaps an input")


@pytest.mark.parametrize("args,words", [
    ((A, -1, 128, B, None, None), "rows"),
    ((A, 4, 0, B, None, None), "columns"),
    ((A, 4, 128, None, None, None), "no output"),
    ((A, 4, 128, None, B, None), "together"),
    ((None, 4, 128, B, None, None), "required"),
    ((A, 4, 128, A + 2046, None, None), "overlaps an input"),
])
def test_silu_mul(lib, args, words):
    refused(lib, "uqm_silu_mul", args, words)


@pytest.mark.parametrize("args,words", [
    ((A, 4, 128, 2, B, C), "blocks"),
    ((A, 4, 128, 0, B, C), "blocks"),
    ((A, -4, 128, 1, B, C), "rows"),
    ((A, 4, 128, 1, None, None), "no output"),
    ((A, 4, 128, 1, B, None), "together"),
    ((None, 4, 128, 1, B, C), "required"),
    ((A, 4, 128, 1, A + 100, C), "overlaps an input"),
])
def test_fp8_quantize(lib, args, words):
    refused(lib, "uqm_fp8_quantize", args, words)


@pytest.mark.parametrize("args,words", [
    ((A, B, -1, C, D, 64, 128, None, E), "rows"),
    ((A, B, 4, C, D, 0, 128, None, E), "features"),
    ((A, B, 4, C, D, 64, 0, None, E), "multiple of 16"),
    ((A, B, 4, C, D, 64, 120, None, E), "multiple of 16"),
    ((A, B, 4, C, D, 64, 1 << 25, None, E), "below 2^25"),
    ((A, B, 4, None, D, 64, 128, None, E), "required"),
    ((A, B, 4, C, None, 64, 128, None, E), "required"),
    ((None, B, 4, C, D, 64, 128, None, E), "required"),
    ((A, None, 4, C, D, 64, 128, None, E), "required"),
    ((A, B, 4, C, D, 64, 128, None, None), "required"),
    ((A + 8, B, 4, C, D, 64, 128, None, E), "aligned"),
    ((A, B, 4, C + 8, D, 64, 128, None, E), "aligned"),
    ((A, B + 2, 4, C, D, 64, 128, None, E), "aligned"),
    ((A, B, 4, C, D, 64, 128, A + 4097, E), "aligned"),
    ((A, B, 4, C, D, 64, 128, None, E + 1), "aligned"),
    ((A, B, 4, C, D, 64, 128, None, A + 510), "overlaps"),
    ((A, B, 4, C, D, 64, 128, E + 2, E), "overlaps"),
])
def test_fp8_linear(lib, args, words):
    refused(lib, "uqm_fp8_linear", args, words)


@pytest.mark.parametrize("args,words", [((-1, 64, 128), "rows"), ((4, 0, 128), "features"), ((4, 64, 8), "multiple of 16")])
def test_fp8_linear_plan(lib, args, words):
    out = [ctypes.byref(ctypes.c_int32()) for _ in range(3)]
    assert lib.uqm_fp8_linear_plan(*args, *out) == 1 and words in lib.uqm_last_error().decode()
    assert lib.uqm_fp8_linear_plan(4, 64, 128, None, *out[1:]) == 1


def test_cases_reach_every_kernel(lib):
    """The GPU tests' sizes (planned for 256 compute units) take the kernels that
    they say, and no size takes another one."""
    assert all(fp8_cases.plan(t, n, k) == kernel for kernel, t, n, k in fp8_cases.PLANNED + fp8_cases.ONE_ROW)
    known = {kernel for kernel, *_ in fp8_cases.PLANNED}
    sizes = [1, 3, 16, 33, 100, 300, 777, 1500, 4000, 9000, 40000]
    assert {fp8_cases.plan(t, n, 16 * k) for t in sizes for n in sizes for k in (1, 8, 40, 128, 600, 600000)} == known


def test_no_rows_is_no_work(lib):
    assert lib.uqm_add_rmsnorm(None, None, 0, 128, None, 1e-6, None, None, None, None, None) == 0
    assert lib.uqm_silu_mul(None, 0, 128, None, None, None, None) == 0
    assert lib.uqm_fp8_quantize(None, 0, 128, 1, None, None, None) == 0
    assert lib.uqm_fp8_linear(None, None, 0, A, B, 64, 128, None, None, None) == 0


# ------------------------------------------------------------- wrappers --
@pytest.fixture(scope="module")
def ext():
    return HipExtension()


def bf(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def fp8(rows, cols, block_rows=1, scales=None):
    groups = -(-cols // 128)
    codes = torch.zeros(rows, cols, dtype=torch.float8_e4m3fn)
    return Fp8Matrix(codes, torch.ones(-(-rows // block_rows), groups) if scales is None else scales, block_rows)


@pytest.mark.parametrize("call,words", [
    (lambda e: e.add_rmsnorm(bf(2, 8).float()), "BF16"),
    (lambda e: e.add_rmsnorm(bf(2, 0)), "column"),
    (lambda e: e.add_rmsnorm(bf(2, 8)), "device tensors"),
    (lambda e: e.add_rmsnorm(bf(2, 8), bf16=False), "at least one"),
    (lambda e: e.add_rmsnorm(bf(2, 8), bf(3, 8)), "hidden's shape"),
    (lambda e: e.add_rmsnorm(bf(2, 8), bf(2, 8).float()), "hidden's shape"),
    (lambda e: e.add_rmsnorm(bf(2, 8), inplace=True), "requires a residual"),
    (lambda e: e.add_rmsnorm(bf(2, 8), bf(8, 2).t(), inplace=True), "contiguous"),
    (lambda e: e.add_rmsnorm(bf(2, 8), weight=bf(7)), "weight"),
    (lambda e: e.add_rmsnorm(bf(2, 8), weight=bf(8).float()), "weight"),
    (lambda e: e.silu_mul(bf(2, 7)), "even"),
    (lambda e: e.silu_mul(bf(2, 8).half()), "BF16"),
    (lambda e: e.silu_mul(bf(2, 8), bf16=False), "at least one"),
    (lambda e: e.silu_mul(bf(2, 8)), "device tensors"),
    (lambda e: e.fp8_quantize(bf(2, 8), block_rows=64), "blocks of 1 or 128"),
    (lambda e: e.fp8_quantize(bf(2, 2, 8), block_rows=128), "matrix"),
    (lambda e: e.fp8_quantize(bf(2, 8).float()), "BF16"),
    (lambda e: e.fp8_linear(fp8(2, 32), fp8(8, 32, 128)), "device tensors"),
    (lambda e: e.fp8_linear(fp8(2, 48), fp8(8, 32, 128)), "input features"),
    (lambda e: e.fp8_linear(bf(2, 48), fp8(8, 32, 128)), "input features"),
    (lambda e: e.fp8_linear(fp8(2, 24), fp8(8, 24, 128)), "multiple of 16"),
    (lambda e: e.fp8_linear(fp8(2, 32), fp8(0, 32, 128)), "at least one row"),
    (lambda e: e.fp8_linear(fp8(2, 32), fp8(8, 32, 1)), "blocks of 128"),
    (lambda e: e.fp8_linear(fp8(128, 32, 128), fp8(8, 32, 128)), "blocks of 1 "),
    (lambda e: e.fp8_linear(fp8(2, 32), fp8(200, 32, 128, torch.ones(1, 1))), "scales"),
    (lambda e: e.fp8_linear(fp8(2, 32, 1, torch.ones(2, 2)), fp8(8, 32, 128)), "scales"),
    (lambda e: e.fp8_linear(fp8(2, 32, 1, torch.ones(2, 1).double()), fp8(8, 32, 128)), "float32 scales"),
    (lambda e: e.fp8_linear(Fp8Matrix(torch.zeros(2, 32, dtype=torch.uint8), torch.ones(2, 1)), fp8(8, 32, 128)),
     "float8_e4m3fn"),
    (lambda e: e.fp8_linear(fp8(2, 32), fp8(8, 32, 128), bf(7)), "bias"),
    (lambda e: e.fp8_linear(fp8(2, 32), fp8(8, 32, 128), bf(8).float()), "bias"),
])
def test_wrappers(ext, call, words):
    with pytest.raises(RuntimeError, match=words):
        call(ext)


@pytest.mark.parametrize("t,n,k", [(1 << 28, 1, 16), ((1 << 31) - 1 - 4096, 1, 16), (1 << 24, 2048, 128), (1, (1 << 31) - 4096, 16),
                                   (1 << 20, 11264, 1 << 23), (1 << 24, 256, (1 << 25) - 16)])
def test_launches_have_room(t, n, k):
    """A launch has less than 2^32 threads."""
    rows, tokens, waves = fp8_cases.plan(t, n, k)
    groups = -(-n // rows) * -(-t // tokens)
    assert -(-groups // 8) * 8 * 64 * waves < 1 << 32


@pytest.mark.parametrize("t,n,k", [((1 << 31) - 1, (1 << 31) - 1, 16), (1, (1 << 31) - 1, 16), ((1 << 31) - 1, 1, 16)])
def test_more_outputs_than_a_launch_has_room_for(lib, t, n, k):
    """2^31 - 1 rows in the largest workgroups: 2^23 of 512 threads, 2^32 threads."""
    got = [ctypes.c_int32() for _ in range(3)]
    assert lib.uqm_fp8_linear_plan(t, n, k, *map(ctypes.byref, got)) == 1
    assert "room" in lib.uqm_last_error().decode()
    refused(lib, "uqm_fp8_linear", (A, B, t, C, D, n, k, None, E), "room")


def test_dequantize_of_a_matrix():
    m = Fp8Matrix(torch.ones(130, 130).to(torch.float8_e4m3fn), torch.tensor([[1.0, 2.0], [3.0, 4.0]]), 128)
    v = m.dequantize()
    assert v.shape == (130, 130) and v[0, 0] == 1 and v[127, 128] == 2 and v[128, 0] == 3 and v[129, 129] == 4
    a = Fp8Matrix(torch.ones(2, 3, 130).to(torch.float8_e4m3fn), torch.arange(12.0).view(2, 3, 2))
    assert a.dequantize()[1, 2, 127] == 10 and a.dequantize()[1, 2, 129] == 11


def test_dense_layers_of_the_host():
    """8-bit dense layers need a HIP device and blocks that run the shared expert
    as a module."""
    from uma_qmoe_amd.formats import ContractError
    from uma_qmoe_amd.qwen_host import load_fixed_qwen, quantize_dense_fp8

    with pytest.raises(ContractError, match="HIP device"):
        load_fixed_qwen("nowhere", "nothing", model_manifest_sha256="0" * 64, device="cpu", fp8_dense=True)
    with pytest.raises(ContractError, match="HIP device"):
        quantize_dense_fp8(torch.nn.Linear(16, 16))


def dense_layer(**changes):
    """A stand-in for a host's layer, BF16 on the CPU."""
    from types import SimpleNamespace

    size = {"q_proj": 32, "k_proj": 32, "v_proj": 32, "o_proj": 32, "gate_proj": 32, "up_proj": 32, "down_proj": 48}
    m = {n: changes.get(n, torch.nn.Linear(k, 32, bias=n in ("q_proj", "k_proj", "v_proj"), dtype=torch.bfloat16)) for n, k in size.items()}
    attn = SimpleNamespace(**{n: m[n] for n in ("q_proj", "k_proj", "v_proj", "o_proj")})
    shared = SimpleNamespace(**{n: m[n] for n in ("gate_proj", "up_proj", "down_proj")})
    return SimpleNamespace(self_attn=attn, mlp=SimpleNamespace(shared_expert=shared, fused_block=changes.get("fused", False)))


@pytest.mark.parametrize("changes,words", [
    ({"fused": True}, "fused_block=False"),
    ({"o_proj": torch.nn.Identity()}, "BF16 Linear"),
    ({"q_proj": torch.nn.Linear(32, 32)}, "BF16 Linear"),
    ({"k_proj": torch.nn.Linear(40, 32, dtype=torch.bfloat16)}, "multiple of 16"),
    ({"down_proj": torch.nn.Linear(24, 32, bias=False, dtype=torch.bfloat16)}, "multiple of 16"),
    ({"up_proj": torch.nn.Linear(32, 32, dtype=torch.bfloat16)}, "no bias"),
    ({"down_proj": torch.nn.Identity()}, "BF16 Linear"),
])
def test_dense_layers_that_stay_as_they_are(changes, words):
    """All layers are looked at before the first is replaced."""
    from uma_qmoe_amd.formats import ContractError
    from uma_qmoe_amd.qwen_host import _check_dense

    _check_dense([dense_layer(), dense_layer()])
    with pytest.raises(ContractError, match=words):
        _check_dense([dense_layer(), dense_layer(**changes)])


def test_dense_layers_with_a_bias_in_fp32():
    """A BF16 weight with an FP32 bias is refused with the model as it was, not by
    every product afterwards."""
    from uma_qmoe_amd.formats import ContractError
    from uma_qmoe_amd.qwen_host import _check_dense

    q_proj = torch.nn.Linear(32, 32, dtype=torch.bfloat16)
    q_proj.bias = torch.nn.Parameter(q_proj.bias.detach().float())
    with pytest.raises(ContractError, match="BF16 bias"):
        _check_dense([dense_layer(), dense_layer(q_proj=q_proj)])


def whole_layer(**changes):
    """A stand-in whose shared expert's projections fit each other."""
    return dense_layer(**{"down_proj": torch.nn.Linear(32, 32, bias=False, dtype=torch.bfloat16), **changes})


def on_hip(*layers):
    """A stand-in for a model whose first parameter is on a HIP device."""
    from types import SimpleNamespace

    return SimpleNamespace(parameters=lambda: iter([SimpleNamespace(device=torch.device("cuda:0"))]),
                           model=SimpleNamespace(layers=layers))


def test_dense_layers_on_the_host():
    """Every projection's device counts, not the first parameter's alone."""
    from uma_qmoe_amd.formats import ContractError
    from uma_qmoe_amd.qwen_host import quantize_dense_fp8

    layers = [whole_layer(), whole_layer()]
    before = [(layer.self_attn.q_proj, layer.mlp.shared_expert) for layer in layers]
    with pytest.raises(ContractError, match="HIP device, layer 0's q_proj is on cpu"):
        quantize_dense_fp8(on_hip(*layers))
    assert all(layer.self_attn.q_proj is q and layer.mlp.shared_expert is s for layer, (q, s) in zip(layers, before))


@pytest.mark.parametrize("changes", [
    {"down_proj": torch.nn.Linear(64, 32, bias=False, dtype=torch.bfloat16)},
    {"gate_proj": torch.nn.Linear(48, 32, bias=False, dtype=torch.bfloat16)},
    {"up_proj": torch.nn.Linear(32, 48, bias=False, dtype=torch.bfloat16)},
])
def test_dense_layers_that_do_not_fit_each_other(changes):
    from uma_qmoe_amd.formats import ContractError
    from uma_qmoe_amd.qwen_host import quantize_dense_fp8

    with pytest.raises(ContractError, match="layer 1's shared expert"):
        quantize_dense_fp8(on_hip(whole_layer(), whole_layer(**changes)))


def test_dense_layers_of_another_activation():
    """The 8-bit shared expert computes SiLU, whatever the module's own function is."""
    from uma_qmoe_amd.formats import ContractError
    from uma_qmoe_amd.qwen_host import quantize_dense_fp8

    layers = [whole_layer(), whole_layer()]
    layers[0].mlp.shared_expert.act_fn = torch.nn.SiLU()
    layers[1].mlp.shared_expert.act_fn = torch.nn.GELU()
    with pytest.raises(ContractError, match="layer 1's shared expert .* SiLU"):
        quantize_dense_fp8(on_hip(*layers))


def test_dense_layers_beside_a_fused_block():
    """A caller who asks for the fused block does not get the other one unsaid."""
    from uma_qmoe_amd.formats import ContractError
    from uma_qmoe_amd.qwen_host import load_fixed_qwen

    with pytest.raises(ContractError, match="fused_block"):
        load_fixed_qwen("nowhere", "nothing", model_manifest_sha256="0" * 64, device="cuda:0", fp8_dense=True, fused_block=True)
