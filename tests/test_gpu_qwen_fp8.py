"""The Qwen host with its dense layers in 8-bit floats: every replaced module
against its definition on the same input, the loaded model against the BF16 one,
and greedy decode replayed from a HIP graph against the same steps run eagerly."""

from __future__ import annotations

import pytest
import torch

import fp8_reference as ref
from qwen_tiny import ARCH, LAYERS, MANIFEST, prompt, write_checkpoint
from uma_qmoe_amd.custom_op import REGISTRY
from uma_qmoe_amd.formats import ContractError
from uma_qmoe_amd.native_backend import install_packed_q4_backend
from uma_qmoe_amd.qwen_host import DecodeGraph, load_fixed_qwen, quantize_dense_fp8

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def checkpoint(tmp_path_factory):
    d = tmp_path_factory.mktemp("qwen_tiny_fp8")
    return d, write_checkpoint(d)[0]


@pytest.fixture(autouse=True)
def _backend():
    install_packed_q4_backend()
    yield
    REGISTRY.uninstall("hip_gfx950")


def load(checkpoint, **kwargs):
    return load_fixed_qwen(*checkpoint, model_manifest_sha256=MANIFEST, device=DEV, performance_mode=True,
                           architecture=ARCH, **kwargs)


def test_modules_compute_their_definition(checkpoint):
    """Each module's inputs are quantised as fp8_quantize does (tested by itself),
    so its product is compared on those codes."""
    print("[case] qwen fp8 modules", flush=True)
    g = torch.Generator().manual_seed(1)
    with load(checkpoint, fp8_dense=True) as host, torch.no_grad():
        assert host.evidence["fp8_dense_weight_count"] == 7 * LAYERS and not host.evidence["fused_block"]
        for layer in host.model.model.layers:
            attn, shared = layer.self_attn, layer.mlp.shared_expert
            for m in (attn.q_proj, attn.k_proj, attn.v_proj, attn.o_proj, shared.gate_up):
                x = torch.randn(2, 3, m.codes.shape[1], generator=g).to(torch.bfloat16).to(DEV)
                q = m.extension.fp8_quantize(x)
                y, tol = ref.linear64(q.codes.view(6, -1), q.scales.view(6, -1), m.codes, m.scales, m.bias)
                assert ((m(x).view(6, -1).double().cpu() - y).abs() <= tol).all()
            x = torch.randn(6, shared.gate_up.codes.shape[1], generator=g).to(torch.bfloat16).to(DEV)
            _, h = shared.down.extension.silu_mul(shared.gate_up(x), bf16=False, fp8=True)
            y, tol = ref.linear64(h.codes, h.scales, shared.down.codes, shared.down.scales, None)
            assert ((shared(x).double().cpu() - y).abs() <= tol).all()


def test_model_is_near_the_bf16_one(checkpoint):
    """An 8-bit product's operands are each off by 2^-4 / sqrt(3) of themselves in
    the mean square at most: 0.051 of its output's norm. Between a hidden state and
    the logits lie, per layer, attention (values, then their projection) and the
    shared expert (two products behind each other), each joining a residual that
    they leave as it is: at most sqrt(4 * LAYERS) * 0.051 = 0.15."""
    print("[case] qwen fp8 model", flush=True)
    ids = prompt(6).to(DEV)
    with torch.no_grad():
        with load(checkpoint, fused_block=False) as host:
            want = host.model(input_ids=ids).logits.float()
        with load(checkpoint, fp8_dense=True) as host:
            got = host.model(input_ids=ids).logits.float()
            one = host.model(input_ids=ids[:, :1]).logits.float()
    assert torch.isfinite(got).all() and torch.isfinite(one).all()
    assert (got - want).norm() <= 0.15 * want.norm()


def test_decode_graph_replays_the_eager_steps(checkpoint):
    print("[case] qwen fp8 decode graph", flush=True)
    ids = prompt(6).to(DEV)
    with load(checkpoint, fp8_dense=True) as host:
        eager, graph = DecodeGraph(host.model, max_len=32), DecodeGraph(host.model, max_len=32)
        assert torch.equal(eager.prefill(ids), graph.prefill(ids))
        graph.capture()
        for i in range(8):
            want, got = eager.step_eager(), graph.replay().clone()
            torch.cuda.synchronize()
            assert torch.equal(got, want), f"token {i}"
            assert (graph.logits - eager.logits).norm() <= 1e-3 * eager.logits.norm(), f"step {i}"


def test_evidence_counts_the_weights_in_8_bits(checkpoint):
    print("[case] qwen fp8 evidence", flush=True)
    with load(checkpoint, fp8_dense=True) as host:
        model = host.model
        held = sum(p.numel() * p.element_size() for p in model.parameters())
        for layer in model.model.layers:
            for m in (*(getattr(layer.self_attn, n) for n in ("q_proj", "k_proj", "v_proj", "o_proj")),
                      layer.mlp.shared_expert.gate_up, layer.mlp.shared_expert.down):
                held += m.codes.numel() + 4 * m.scales.numel() + (0 if m.bias is None else 2 * m.bias.numel())
        assert host.evidence["model_parameter_bytes"] == held


def test_a_second_call_is_refused(checkpoint):
    print("[case] qwen fp8 twice", flush=True)
    ids = prompt(3).to(DEV)
    with load(checkpoint, fp8_dense=True) as host, torch.no_grad():
        want = host.model(input_ids=ids).logits
        with pytest.raises(ContractError, match="BF16 Linear"):
            quantize_dense_fp8(host.model)
        assert (host.model(input_ids=ids).logits - want).norm() <= 1e-3 * want.norm()
