"""Batched greedy decode over a paged cache: each sequence as it is decoded alone
by ``DecodeGraph``, and the replays of a captured step as the same steps run eagerly."""

from __future__ import annotations

import pytest
import torch

from oracle import moe as om
from qwen_tiny import ARCH, MANIFEST, prompt, write_checkpoint
from uma_qmoe_amd.custom_op import REGISTRY
from uma_qmoe_amd.formats import ContractError
from uma_qmoe_amd.native_backend import install_packed_q4_backend
from uma_qmoe_amd.paged_decode import PagedDecodeGraph
from uma_qmoe_amd.qwen_host import DecodeGraph, load_fixed_qwen

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def checkpoint(tmp_path_factory):
    d = tmp_path_factory.mktemp("qwen_tiny_paged")
    return d, write_checkpoint(d)[0]


@pytest.fixture(autouse=True)
def _backend():
    install_packed_q4_backend()
    yield
    REGISTRY.uninstall("hip_gfx950")


def load(checkpoint, **kwargs):
    return load_fixed_qwen(*checkpoint, model_manifest_sha256=MANIFEST, device=DEV, performance_mode=True,
                           architecture=ARCH, **kwargs)


def uncached(model, ids):
    with torch.no_grad():
        return model(input_ids=ids).logits[0, -1].float()


# Logits of a step against the whole sequence run again: BF16 as the one-sequence
# graph's test allows (2e-2). An 8-bit cache's keys and values are each off by at most
# 2^-4 of themselves, in the mean square 2^-4 / sqrt(3) = 0.036 at most: per layer
# sqrt(2) * 0.036 of what attention adds, over LAYERS = 2 layers 0.072, beside the 2e-2.
LIMIT = {False: 2e-2, True: 9.2e-2}


@pytest.mark.parametrize("fp8", [False, True])
def test_sequences_of_a_batch_are_those_decoded_alone(checkpoint, fp8):
    """Every step's logits against the sequence run again without a cache, on the
    tokens that the batch chose; a page ends in the middle of the decode."""
    print(f"[case] paged decode {fp8}", flush=True)
    prompts = [prompt(n, seed=n).to(DEV) for n in (6, 1, 13)]
    with load(checkpoint) as host:
        dg = PagedDecodeGraph(host.model, batch=4, max_len=48, page_size=16, fp8_cache=fp8)
        seqs = []
        for i, ids in zip((0, 2, 3), prompts):
            seqs.append((i, torch.cat([ids, dg.prefill(i, ids)], 1)))
            assert om.rel_l2(dg.token[i].float().cpu(), seqs[-1][1][0, -1:].float().cpu()) == 0
        for step in range(12):
            got = dg.step_eager()
            for n, (i, ids) in enumerate(seqs):
                r = om.rel_l2(dg.logits[i].cpu(), uncached(host.model, ids).cpu())
                assert r <= LIMIT[fp8], f"step {step}, sequence {i}: rel-L2 {r}"
                seqs[n] = (i, torch.cat([ids, got[i:i + 1]], 1))


@pytest.mark.parametrize("fp8", [False, True])
def test_replays_are_the_eager_steps(checkpoint, fp8):
    """Also when sequences end and begin between replays."""
    print(f"[case] paged replays {fp8}", flush=True)
    prompts = [prompt(n, seed=n).to(DEV) for n in (6, 15, 2)]
    with load(checkpoint) as host:
        eager, graph = (PagedDecodeGraph(host.model, batch=3, max_len=64, page_size=16, fp8_cache=fp8) for _ in range(2))
        for dg in (eager, graph):
            dg.prefill(0, prompts[0])
            dg.prefill(1, prompts[1])
        graph.capture()
        for step in range(20):
            if step == 6:
                for dg in (eager, graph):
                    dg.finish(0)
                    dg.prefill(2, prompts[2])
            if step == 11:
                for dg in (eager, graph):
                    dg.prefill(0, prompts[1])
            live = [i for i in range(3) if eager.next_positions[i] is not None]
            want, got = eager.step_eager(), graph.replay().clone()
            torch.cuda.synchronize()
            assert torch.equal(got[live], want[live]), f"step {step}"
            assert (graph.logits[live] - eager.logits[live]).norm() <= 1e-3 * eager.logits[live].norm(), f"step {step}"
        assert graph.next_positions == eager.next_positions == [15 + 9, 15 + 20, 2 + 14]


def test_with_dense_layers_in_8_bits(checkpoint):
    """A host whose projections are 8-bit modules: replays are the eager steps."""
    print("[case] paged fp8 dense", flush=True)
    with load(checkpoint, fp8_dense=True) as host:
        eager, graph = (PagedDecodeGraph(host.model, batch=2, max_len=40, page_size=16, fp8_cache=True) for _ in range(2))
        for dg in (eager, graph):
            dg.prefill(0, prompt(5, seed=1).to(DEV))
            dg.prefill(1, prompt(17, seed=2).to(DEV))
        graph.capture()
        for step in range(8):
            want, got = eager.step_eager(), graph.replay().clone()
            torch.cuda.synchronize()
            assert torch.equal(got, want), f"step {step}"
            assert (graph.logits - eager.logits).norm() <= 1e-3 * eager.logits.norm(), f"step {step}"


def test_one_sequence_is_the_one_sequence_graph(checkpoint):
    """The same logits as DecodeGraph's, from a captured step each, as long as both
    choose the same tokens. Either is within 2e-2 of the sequence run again without a
    cache (as the tests of each require), so they are within 2 * 2e-2 / (1 - 2e-2) of
    each other: 4.1e-2. (2e-2 was asked for at first, which one of 16 steps passed by
    3e-3.)"""
    print("[case] paged against static cache", flush=True)
    ids = prompt(9).to(DEV)
    with load(checkpoint) as host:
        a, b = DecodeGraph(host.model, max_len=40), PagedDecodeGraph(host.model, batch=1, max_len=40, page_size=16)
        assert torch.equal(a.prefill(ids), b.prefill(0, ids))
        a.capture()
        b.capture()
        for step in range(16):
            x, y = a.replay().clone(), b.replay().clone()
            torch.cuda.synchronize()
            assert om.rel_l2(b.logits[0].cpu(), a.logits.cpu()) <= 4.1e-2, f"step {step}"
            if not torch.equal(x, y):
                break
        assert step > 0


@pytest.mark.parametrize("fp8", [False, True])
def test_a_conversation_goes_on(checkpoint, fp8):
    """Tokens added to a sequence attend to what the cache holds of it."""
    print(f"[case] paged extend {fp8}", flush=True)
    with load(checkpoint) as host:
        dg = PagedDecodeGraph(host.model, batch=2, max_len=96, page_size=32, fp8_cache=fp8)
        seq = torch.cat([prompt(20, seed=1).to(DEV), dg.prefill(1, prompt(20, seed=1).to(DEV))], 1)
        for _ in range(5):
            seq = torch.cat([seq, dg.step_eager()[1:]], 1)
        more = torch.cat([seq[:, -1:], prompt(17, seed=2).to(DEV)], 1)  # the last choice and the next turn
        seq = torch.cat([seq[:, :-1], more], 1)
        assert torch.equal(dg.extend(1, more), dg.token[1:])
        seq = torch.cat([seq, dg.token[1:]], 1)
        for step in range(4):
            want = uncached(host.model, seq)
            seq = torch.cat([seq, dg.step_eager()[1:]], 1)
            assert om.rel_l2(dg.logits[1].cpu(), want.cpu()) <= LIMIT[fp8], f"step {step}"


@pytest.mark.parametrize("fp8", [False, True])
def test_a_layer_with_a_window(checkpoint, fp8):
    """A layer that sees the last 8 positions only: in prefill, in steps and when a conversation goes on."""
    print(f"[case] paged window {fp8}", flush=True)
    with load(checkpoint) as host:
        host.model.config.layer_types = ["full_attention", "sliding_attention"]
        host.model.config.sliding_window = 8
        host.model.model.layers[1].self_attn.sliding_window = 8
        dg = PagedDecodeGraph(host.model, batch=1, max_len=96, page_size=16, fp8_cache=fp8)
        ids = prompt(21, seed=5).to(DEV)
        seq = torch.cat([ids, dg.prefill(0, ids)], 1)
        for step in range(6):
            want = uncached(host.model, seq)
            seq = torch.cat([seq, dg.step_eager()], 1)
            assert om.rel_l2(dg.logits[0].cpu(), want.cpu()) <= LIMIT[fp8], f"step {step}"
        seq = torch.cat([seq, prompt(9, seed=6).to(DEV)], 1)
        dg.extend(0, seq[:, dg.next_positions[0]:])  # (the last choice and what follows)
        seq = torch.cat([seq, dg.token], 1)
        want = uncached(host.model, seq)
        dg.step_eager()
        assert om.rel_l2(dg.logits[0].cpu(), want.cpu()) <= LIMIT[fp8]
        # (the window matters: a model without it gives other logits)
        host.model.config.layer_types = ["full_attention", "full_attention"]
        assert om.rel_l2(want.cpu(), uncached(host.model, seq).cpu()) > LIMIT[fp8]


def test_refusals_change_nothing(checkpoint):
    print("[case] paged refusals", flush=True)
    ids = prompt(10).to(DEV)
    with load(checkpoint) as host:
        for kwargs, words in ((dict(batch=0, max_len=8), "at least one"), (dict(batch=1, max_len=0), "at least one"),
                              (dict(batch=1, max_len=8, page_size=24), "pages of")):
            with pytest.raises(ContractError, match=words):
                PagedDecodeGraph(host.model, **kwargs)
        host.model.config.model_type = "olmoe"
        with pytest.raises(ContractError, match="Qwen2MoE"):
            PagedDecodeGraph(host.model, batch=1, max_len=8)
        host.model.config.model_type = "qwen2_moe"
        dg = PagedDecodeGraph(host.model, batch=2, max_len=20, page_size=16, pages=2)
        with pytest.raises(ContractError, match="no sequence"):
            dg.step_eager()
        with pytest.raises(ContractError, match="capture"):
            dg.replay()
        for bad in (-1, 2):
            with pytest.raises(ContractError, match="no place"):
                dg.prefill(bad, ids)
        for n in (0, 20):
            with pytest.raises(ContractError, match="prompt must"):
                dg.prefill(0, prompt(max(n, 1)).to(DEV)[:, :n])
        dg.prefill(0, ids)
        dg.prefill(1, ids)
        with pytest.raises(ContractError, match="shorter than the cache"):
            dg.extend(0, ids)
        for _ in range(6):
            dg.step_eager()
        before = (dg.token.clone(), dg.positions.clone(), dg.page_table.clone(), list(dg.next_positions))
        with pytest.raises(ContractError, match="0 free pages, 2 are needed"):
            dg.step_eager()
        assert torch.equal(dg.token, before[0]) and torch.equal(dg.positions, before[1])
        assert torch.equal(dg.page_table, before[2]) and dg.next_positions == before[3]
        with pytest.raises(ContractError, match="0 free pages, 1 are needed"):
            dg.prefill(0, prompt(17).to(DEV))
        assert dg.next_positions == before[3]
        dg.finish(0)
        for _ in range(4):
            dg.step_eager()  # with the page that the other sequence had
        with pytest.raises(ContractError, match=r"sequences \[1\] have filled their places"):
            dg.step_eager()
