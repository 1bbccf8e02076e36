"""What a decode object holds between its calls: eager steps and replays mixed on one
object, and calls that fail or are refused with the sequences left as they were."""

from __future__ import annotations

import sys

import pytest
import torch

from oracle import moe as om
from qwen_tiny import prompt
from test_gpu_paged_decode import DEV, _backend, checkpoint, load  # noqa: F401 (fixtures)
from uma_qmoe_amd.formats import ContractError
from uma_qmoe_amd.native_backend import load_native_extension
from uma_qmoe_amd.paged_decode import PagedDecodeGraph
from uma_qmoe_amd.qwen_host import DecodeGraph

pytestmark = pytest.mark.gpu


def same(a, b, what):
    assert torch.equal(a.token, b.token), what
    assert (a.logits - b.logits).norm() <= 1e-3 * b.logits.norm(), what


def mixed_steps(mixed, eager):
    """Eager steps, a capture and replays on one object, eager steps on the other."""
    for step, kind in enumerate(["step_eager", "step_eager", "capture", "replay", "replay", "step_eager", "replay", "capture",
                                 "replay", "step_eager", "step_eager", "capture", "step_eager", "replay", "replay"]):
        if kind == "capture":
            held = mixed.logits.clone()
            mixed.capture()
            torch.cuda.synchronize()
            assert torch.equal(mixed.logits, held), "capturing is no step"
            continue
        getattr(mixed, kind)()
        eager.step_eager()
        torch.cuda.synchronize()
        same(mixed, eager, f"{kind} {step}")


@pytest.mark.parametrize("fp8", [False, True])
def test_logits_are_the_last_steps(checkpoint, fp8):
    print(f"[case] paged logits {fp8}", flush=True)
    with load(checkpoint) as host:
        mixed, eager = (PagedDecodeGraph(host.model, batch=2, max_len=64, page_size=16, fp8_cache=fp8) for _ in range(2))
        for dg in (mixed, eager):
            dg.prefill(0, prompt(5, seed=1).to(DEV))
            dg.prefill(1, prompt(17, seed=2).to(DEV))
        mixed_steps(mixed, eager)


def test_logits_of_a_capture_before_the_first_step(checkpoint):
    print("[case] paged logits before a step", flush=True)
    with load(checkpoint) as host:
        dg = PagedDecodeGraph(host.model, batch=1, max_len=32)
        dg.prefill(0, prompt(5, seed=1).to(DEV))
        dg.capture()
        assert dg.logits is None
        dg.replay()
        assert dg.logits.isfinite().all()


def test_logits_of_the_one_sequence_graph_are_the_last_steps(checkpoint):
    print("[case] static logits", flush=True)
    with load(checkpoint) as host:
        mixed, eager = (DecodeGraph(host.model, max_len=64) for _ in range(2))
        for dg in (mixed, eager):
            dg.prefill(prompt(9).to(DEV))
        mixed_steps(mixed, eager)


def state(dg):
    return (dg.page_table.tolist(), dg.positions.tolist(), dg.lengths.tolist(), dg.active.tolist(), dg.token.tolist(),
            list(dg.next_positions), [list(o) for o in dg.pool.owned], list(dg.pool.free))


def pair(host, **kwargs):
    """Two objects with the same two sequences of three places."""
    objects = [PagedDecodeGraph(host.model, batch=3, max_len=64, page_size=16, **kwargs) for _ in range(2)]
    for dg in objects:
        dg.prefill(0, prompt(5, seed=1).to(DEV))
        dg.prefill(2, prompt(15, seed=2).to(DEV))
        for _ in range(3):
            dg.step_eager()
    return objects


@pytest.mark.parametrize("bad", [
    torch.ones(2, 4, dtype=torch.long), torch.ones(4, dtype=torch.long), torch.ones(1, 2, 2, dtype=torch.long),
    torch.ones(1, 4), torch.ones(1, 4, dtype=torch.bool)])
def test_tokens_of_another_form_are_refused(checkpoint, bad):
    """Before anything of the sequence is given up."""
    print(f"[case] paged tokens {tuple(bad.shape)} {bad.dtype}", flush=True)
    with load(checkpoint) as host:
        dg, twin = pair(host)
        before = state(dg)
        for call in (dg.prefill, dg.extend):
            for ids in (bad.to(DEV), torch.ones(1, 4, dtype=torch.long)):  # (also on the host)
                with pytest.raises(ContractError, match="token ids"):
                    call(2, ids)
                assert state(dg) == before
        for _ in range(3):
            dg.step_eager()
            twin.step_eager()
            same_sequences(dg, twin)


def same_sequences(a, b, live=(0, 2)):
    live = list(live)
    assert torch.equal(a.token[live], b.token[live])
    assert (a.logits[live] - b.logits[live]).norm() <= 1e-3 * b.logits[live].norm()


def failing(host, layer):
    """A model whose ``layer`` runs out of memory."""
    def fail(*_):
        raise RuntimeError("out of memory")
    return host.model.model.layers[layer].mlp.register_forward_pre_hook(fail)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("layer", [0, 1])
def test_tokens_that_could_not_be_added(checkpoint, layer, fp8):
    """The model fails: the sequence is as it was, and its pages are those it had."""
    print(f"[case] paged extend fails {layer} {fp8}", flush=True)
    more = prompt(20, seed=3).to(DEV)
    with load(checkpoint) as host:
        dg, twin = pair(host, fp8_cache=fp8)
        before = state(dg)
        hook = failing(host, layer)
        with pytest.raises(RuntimeError, match="out of memory"):
            dg.extend(2, more)
        hook.remove()
        assert state(dg) == before
        for _ in range(3):
            dg.step_eager()
            twin.step_eager()
            same_sequences(dg, twin)
        for x in (dg, twin):
            x.extend(2, more)
            x.step_eager()
        same_sequences(dg, twin)


def test_a_prompt_that_could_not_be_put_in(checkpoint):
    """The model fails: the place is empty, and the pool has all of its pages."""
    print("[case] paged prefill fails", flush=True)
    ids = prompt(20, seed=3).to(DEV)
    with load(checkpoint) as host:
        dg, twin = pair(host)
        for place in (1, 2):  # an empty one, and one with a sequence (which ends)
            hook = failing(host, 1)
            with pytest.raises(RuntimeError, match="out of memory"):
                dg.prefill(place, ids)
            hook.remove()
            assert dg.pool.owned[place] == [] and dg.next_positions[place] is None
            assert sorted(dg.pool.free + dg.pool.owned[0] + dg.pool.owned[2]) == list(range(12))
            assert dg.page_table[place].eq(-1).all() and dg.lengths[place] == 0 and dg.active[place] == 0
        twin.finish(2)
        dg.step_eager()
        twin.step_eager()
        same_sequences(dg, twin, [0])
        for x in (dg, twin):
            x.prefill(2, ids)
            x.step_eager()
        same_sequences(dg, twin)


def test_tokens_for_no_sequence_are_refused(checkpoint):
    """A sequence that has ended does not go on as a new one."""
    print("[case] paged extend of nothing", flush=True)
    with load(checkpoint) as host:
        dg, _ = pair(host)
        dg.finish(2)
        before = state(dg)
        for place in (1, 2):
            with pytest.raises(ContractError, match=f"no sequence at {place}"):
                dg.extend(place, prompt(4).to(DEV))
            assert state(dg) == before


@pytest.mark.parametrize("paged", [True, False])
def test_a_capture_waits_for_its_own_device(checkpoint, monkeypatch, paged):
    """The work before a capture is on the model's device, whichever is the current one."""
    print(f"[case] capture's stream {paged}", flush=True)
    asked, current = [], torch.cuda.current_stream

    def recorded(device=None):
        if sys._getframe(1).f_code.co_filename.endswith(("paged_decode.py", "qwen_host.py")):
            asked.append(device)
        return current(device)

    with load(checkpoint) as host:
        if paged:
            dg = PagedDecodeGraph(host.model, batch=1, max_len=32)
            dg.prefill(0, prompt(5).to(DEV))
        else:
            dg = DecodeGraph(host.model, max_len=32)
            dg.prefill(prompt(5).to(DEV))
        monkeypatch.setattr(torch.cuda, "current_stream", recorded)
        dg.capture()
        assert asked and all(d == dg.device for d in asked)


def test_the_same_tokens_in_both_caches(checkpoint):
    """Every step of DecodeGraph and PagedDecodeGraph on the same tokens: either's logits are
    within 2e-2 of the sequence run again without a cache, so within 2 * 2e-2 / (1 - 2e-2) of
    each other, and a choice differs only where the two best logits are closer than that."""
    print("[case] paged and static cache, same tokens", flush=True)
    limit = 4.1e-2
    ids = prompt(9).to(DEV)
    with load(checkpoint) as host:
        a, b = DecodeGraph(host.model, max_len=40), PagedDecodeGraph(host.model, batch=1, max_len=40, page_size=16)
        a.prefill(ids)
        b.prefill(0, ids)
        b.token.copy_(a.token)
        a.capture()
        b.capture()
        for step in range(24):
            a.replay()
            b.replay()
            torch.cuda.synchronize()
            x, y = a.logits.double().cpu(), b.logits[0].double().cpu()
            assert om.rel_l2(y, x) <= limit, f"step {step}"
            if not torch.equal(a.token, b.token):
                # (each logit is off by no more than the whole difference's norm)
                assert x.max() - x[int(b.token)] <= 2 * (y - x).norm(), f"step {step}"
            b.token.copy_(a.token)


@pytest.mark.parametrize("paged", [True, False])
def test_a_graph_keeps_its_workspace(checkpoint, paged):
    """A larger call on the capture's stream between replays, and memory that is filled
    afterwards: replays are the eager steps."""
    print(f"[case] captured workspace {paged}", flush=True)
    with load(checkpoint) as host:
        graph, eager = ((PagedDecodeGraph(host.model, batch=1, max_len=64, page_size=16) if paged else
                         DecodeGraph(host.model, max_len=64)) for _ in range(2))
        for dg in (graph, eager):
            dg.prefill(*((0, prompt(9).to(DEV)) if paged else (prompt(9).to(DEV),)))
        graph.capture()
        for n in (30, 100):
            graph.replay()
            eager.step_eager()
            graph.stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(graph.stream), torch.no_grad():
                host.model(input_ids=prompt(n).to(DEV))
                filled = [torch.full((m,), 255, dtype=torch.uint8, device=DEV) for m in (1 << 12, 1 << 16, 1 << 18, 1 << 20) for _ in range(8)]
            torch.cuda.current_stream().wait_stream(graph.stream)
            graph.replay()
            eager.step_eager()
            torch.cuda.synchronize()
            same(graph, eager, f"{n}")
            assert all(t.eq(255).all() for t in filled)
        load_native_extension()[1].status()
