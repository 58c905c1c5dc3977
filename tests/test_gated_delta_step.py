"""The gated delta rule's single-token step (gated_delta_state_update) against the formula in 64 bits, and a prompt followed by steps against
one whole sequence.

Tolerances, relative to the largest value compared: fp32 arithmetic over dk <= 128 terms, twice: 2 * 128 * 2^-24 = 1.5e-5 at worst; what is stored
in 16 bits adds one rounding (2^-8 bf16, 2^-11 fp16); inputs are exact."""
import pytest
import torch

from mamba_ssm.ops.gated_delta_rule import (gated_delta_rule_fn, gated_delta_state_update, gated_delta_state_update_ref)
from test_gated_delta import DTYPES, TOL, close, inputs

STORED = {torch.float32: 1.5e-5, torch.float16: 1.5e-5 + 2**-11, torch.bfloat16: 1.5e-5 + 2**-8}


def step_inputs(b, hk, h, dk, dv, dtype, state_dtype=torch.float32, seed=0, device="cuda", gate_dtype=None):
    t = {k: v[:, 0] for k, v in inputs(b, 1, hk, h, dk, dv, dtype, seed=seed, device=device, gate_dtype=gate_dtype).items()}
    r = torch.Generator(device=device).manual_seed(seed + 50)
    return torch.randn(b, h, dk, dv, generator=r, device=device).to(state_dtype), t


def check(state, t, scale=None):
    want_state = state.double()
    want = gated_delta_state_update_ref(want_state, **{k: v.double() for k, v in t.items()}, scale=scale)
    got = gated_delta_state_update(state, **t, scale=scale)
    assert got.dtype == t["v"].dtype and got.shape == t["v"].shape
    close(got, want, STORED[t["v"].dtype], "out")
    close(state, want_state, STORED[state.dtype], "state")


@pytest.mark.parametrize("change, message", [
    (lambda s, t: (s[:, :, :3], t), "state must be"),
    (lambda s, t: (s.double(), t), "state must be"),
    (lambda s, t: (s, {**t, "q": t["q"][..., :2]}), "expected"),
    (lambda s, t: (s, {**t, "v": t["v"].half()}), "one dtype"),
    (lambda s, t: (s, {**t, "beta": t["beta"][:, :1]}), "shape of v"),
    (lambda s, t: (s, t), "GPU"),
])
def test_refusals(change, message):
    state, t = step_inputs(2, 1, 2, 4, 6, torch.float32, device="cpu")
    state, t = change(state, t)
    with pytest.raises(RuntimeError, match=message):
        gated_delta_state_update(state, **t)


def test_sizes_beyond_32_bits_are_refused():
    state, t = step_inputs(1, 1, 1, 4, 6, torch.float32, device="cpu")
    with pytest.raises(RuntimeError, match="2\\^31"):
        gated_delta_state_update(state, **{k: v.expand(2**32 + 3, *v.shape[1:]) for k, v in t.items()})


def test_states_must_stand_apart():
    from mamba_ssm.ops.gated_delta_rule import _separate_states
    s = torch.zeros(3, 2, 4, 5)
    assert _separate_states(s) and _separate_states(s.transpose(0, 1)) and _separate_states(s[::2]) and _separate_states(s[:1].expand(1, 2, 4, 5))
    assert not _separate_states(s[:1].expand(3, 2, 4, 5)) and not _separate_states(s.transpose(2, 3)) and not _separate_states(s[..., :3])
    assert not _separate_states(torch.zeros(100).as_strided((2, 2, 4, 5), (10, 20, 5, 1)))


def test_c_entry_refuses():
    import ctypes

    import vms_hip
    L = vms_hip.lib()
    P = vms_hip.GatedDeltaStepParams()
    assert L.vms_gated_delta_state_update(None, None) < 0
    assert L.vms_gated_delta_state_update(ctypes.byref(P), None) < 0 and b"empty" in L.vms_last_error()
    P.batch = P.heads = P.heads_k = 1
    P.dk, P.dv = 129, 4
    assert L.vms_gated_delta_state_update(ctypes.byref(P), None) < 0 and b"key heads" in L.vms_last_error()
    P.dk = 4
    assert L.vms_gated_delta_state_update(ctypes.byref(P), None) < 0 and b"required" in L.vms_last_error()


def test_c_entry_refuses_launches_of_2_to_the_32_threads():
    import ctypes

    import vms_hip
    L = vms_hip.lib()
    P = vms_hip.GatedDeltaStepParams()
    P.heads, P.heads_k, P.dk, P.dv = 2**8, 1, 4, 40   # two workgroups of 256 threads per head
    for batch, message in ((2**15, b"too large"), (2**15 - 1, b"required")):
        P.batch = batch
        assert L.vms_gated_delta_state_update(ctypes.byref(P), None) < 0 and message in L.vms_last_error(), L.vms_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b, hk, h, dk, dv", [(1, 1, 1, 1, 1), (3, 2, 4, 5, 7), (2, 1, 1, 32, 33), (1, 8, 8, 128, 128), (2, 2, 6, 40, 72),
                                              (5, 1, 2, 64, 30), (2, 3, 3, 100, 130), (70, 4, 8, 65, 31)])
def test_step(b, hk, h, dk, dv, dtype):
    check(*step_inputs(b, hk, h, dk, dv, dtype, seed=dk))


@pytest.mark.gpu
@pytest.mark.parametrize("state_dtype", DTYPES)
def test_state_types_and_gates(state_dtype):
    state, t = step_inputs(2, 2, 4, 48, 52, torch.bfloat16, state_dtype, gate_dtype=torch.float32)
    check(state, t, scale=0.3)
    t["g"][:] = float("-inf")   # all forgotten, however large the state was
    state.fill_(1e4)
    check(state, t)
    t["beta"][:] = 0
    t["g"][:] = 0   # nothing happens to the state
    before = state.clone()
    gated_delta_state_update(state, **t)
    assert torch.equal(before, state)


@pytest.mark.gpu
def test_step_strides():
    """a pool's states seen as (batch, heads), odd offsets, heads before batch, inputs cut from a fused projection"""
    state, t = step_inputs(3, 2, 2, 24, 20, torch.bfloat16)
    a = state.clone()
    want = gated_delta_state_update(a, **t)
    b = state.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(want, gated_delta_state_update(b, **t)) and torch.equal(a, b)
    buf = torch.zeros(2 * state.numel() + 1, device="cuda")
    c = buf[1:].view(6, 2, 24, 20)[::2]
    c.copy_(state)
    fused = torch.cat([x.flatten(1) for x in (t["q"], t["k"], t["v"])], -1)
    q, k, v = fused.split([48, 48, 40], -1)
    assert torch.equal(want, gated_delta_state_update(c, q.view(3, 2, 24), k.view(3, 2, 24), v.view(3, 2, 20), t["g"], t["beta"]))
    assert torch.equal(a, c) and (buf[1:].view(6, 2, 24, 20)[1::2] == 0).all() and buf[0] == 0
    strided = {n: torch.stack([x, x], -1)[..., 0] for n, x in t.items()}
    d = state.clone()
    assert torch.equal(want, gated_delta_state_update(d, **strided)) and torch.equal(a, d)


@pytest.mark.gpu
def test_step_refuses_overlap_and_gradients():
    state, t = step_inputs(3, 1, 1, 8, 8, torch.float32)
    with pytest.raises(RuntimeError, match="overlap"):
        gated_delta_state_update(state[:1].expand(3, -1, -1, -1), **t)
    with pytest.raises(RuntimeError, match="gradient"):
        gated_delta_state_update(state, **{**t, "v": t["v"].clone().requires_grad_()})
    with torch.no_grad():
        gated_delta_state_update(state, **t)
    empty = gated_delta_state_update(state[:0], **{n: x[:0] for n, x in t.items()})
    assert empty.shape == (0, 1, 8)


@pytest.mark.gpu
def test_step_captured():
    state, t = step_inputs(2, 2, 2, 64, 64, torch.bfloat16)
    ref = state.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        gated_delta_state_update(state.clone(), **t)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = gated_delta_state_update(state, **t)
    for _ in range(3):
        graph.replay()
        want = gated_delta_state_update(ref, **t)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(state, ref)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_prompt_then_steps(dtype):
    """a prompt by gated_delta_rule_fn, the rest token by token, against the whole sequence in one call"""
    t = inputs(2, 90, 2, 4, 64, 48, dtype, seed=4)
    whole, final = gated_delta_rule_fn(**t, return_final_state=True)
    out, state = gated_delta_rule_fn(**{k: v[:, :75] for k, v in t.items()}, return_final_state=True)
    rest = [gated_delta_state_update(state, **{k: v[:, i] for k, v in t.items()}) for i in range(75, 90)]
    close(torch.cat([out, torch.stack(rest, 1)], 1), whole, 2 * TOL[dtype])
    close(state, final, 4e-4 if dtype != torch.float32 else 4e-5)


@pytest.mark.gpu
def test_compiled_and_ctypes_steps_are_one(monkeypatch):
    import vms_hip
    ext = vms_hip.ext()
    assert ext is not None
    state, t = step_inputs(2, 2, 4, 40, 48, torch.float16, torch.float16)
    runs = []
    for use in (ext, None):
        monkeypatch.setattr(vms_hip, "_ext", use)
        s = state.clone()
        version = s._version
        runs.append([gated_delta_state_update(s, **t), s, gated_delta_state_update(s.clone(), **t, scale=0.25)])
        assert s._version > version   # autograd sees the update
        for bad in (state.transpose(2, 3), state[:1].expand(2, -1, -1, -1), state.double(), state.cpu()):
            with pytest.raises(RuntimeError, match="gated_delta_rule"):
                gated_delta_state_update(bad, **t)
    assert all(torch.equal(a, b) for a, b in zip(*runs))


@pytest.mark.gpu
@pytest.mark.parametrize("compiled", [True, False])
def test_state_of_an_inference_mode(compiled, monkeypatch):
    """a prompt worked under inference_mode, steps outside of it: the state of such a call counts no versions and is updated like any other"""
    import vms_hip
    if not compiled:
        monkeypatch.setattr(vms_hip, "_ext", None)
    state, t = step_inputs(2, 1, 2, 16, 20, torch.bfloat16)
    want_state = state.clone()
    with torch.inference_mode():
        inner = state.clone()
    for _ in range(2):
        want = gated_delta_state_update(want_state, **t)
        with torch.no_grad():
            got = gated_delta_state_update(inner, **t)
        assert torch.equal(got, want) and torch.equal(inner, want_state)
    with torch.inference_mode():
        assert torch.equal(gated_delta_state_update(inner, **t), gated_delta_state_update(want_state, **t))
