"""Gated delta rule (mamba_ssm.ops.gated_delta_rule) against its recurrence in 64 bits.

Tolerances, relative to the largest value of the tensor compared (fixed before the first run):
  outputs and gradients in bf16 / fp16: a value passes at most six roundings to that type (an input of a product, a stored state or
    intermediate, the result; eps / 2 = 2^-8, 2^-11 each): 6 * 2^-8 = 2.4e-2, 6 * 2^-11 = 2.9e-3;
  fp32 states beside 16-bit inputs: operands are two bf16 planes, each product is off by at most 3 * 2^-16 (two residuals, one product of
    residuals left out), and four products stand in a row from one chunk's state to the next: 12 * 2^-16 = 1.8e-4;
  fp32: operands are exact (three planes); sums of up to 128 + 64 terms in a row in fp32, random signs: well under 2e-5."""
import math

import pytest
import torch

from mamba_ssm.ops.gated_delta_rule import gated_delta_rule_fn, gated_delta_rule_ref

TOL = {torch.float32: 2e-5, torch.float16: 6 * 2**-11, torch.bfloat16: 6 * 2**-8}
STATE_TOL = {torch.float32: 2e-5, torch.float16: 12 * 2**-16, torch.bfloat16: 12 * 2**-16}


def close(got, want, tol, what=""):
    want = want.double()
    top = want.abs().max().item() if want.numel() else 0.0
    off = (got.double() - want).abs().max().item() if want.numel() else 0.0
    assert off <= tol * max(top, 1e-30), f"{what}: off by {off:.3e} of {top:.3e} ({off / max(top, 1e-30):.2e} > {tol:.2e})"


def inputs(b, l, hk, h, dk, dv, dtype, state=False, seed=0, device="cuda", gate_dtype=None):
    r = torch.Generator(device=device).manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=r, device=device)  # noqa: E731
    unit = lambda x: x / x.norm(dim=-1, keepdim=True).clamp_min(1e-6)  # noqa: E731
    gd = gate_dtype or dtype
    t = {"q": unit(randn(b, l, hk, dk)).to(dtype), "k": unit(randn(b, l, hk, dk)).to(dtype), "v": randn(b, l, h, dv).to(dtype),
         "g": (-2 * torch.nn.functional.softplus(randn(b, l, h) - 3)).to(gd), "beta": torch.sigmoid(randn(b, l, h)).to(gd)}
    if state:
        t["initial_state"] = 0.3 * randn(b, h, dk, dv)
    return t


def both(t, dout, dfinal=None, **kw):
    """(out, final, gradients) of the kernels and of the recurrence in 64 bits on the same values"""
    res = []
    for fn, cast in ((gated_delta_rule_fn, lambda x: x.detach().clone()), (gated_delta_rule_ref, lambda x: x.detach().double())):
        leaf = {k: cast(v).requires_grad_() for k, v in t.items()}
        out, final = fn(**leaf, return_final_state=True, **kw)
        heads = [(out, dout.to(out.dtype))] + ([(final, dfinal.to(final.dtype))] if dfinal is not None else [])
        grads = torch.autograd.grad([x for x, _ in heads], list(leaf.values()), [g for _, g in heads])
        res.append((out, final, dict(zip(leaf, grads))))
    return res


def compare(t, seed=1, final_grad=True, **kw):
    dtype = t["v"].dtype
    r = torch.Generator(device=t["v"].device).manual_seed(seed)
    dout = torch.randn(t["v"].shape, generator=r, device=t["v"].device).to(dtype)
    b, l, h, dv = t["v"].shape
    dfinal = 0.3 * torch.randn(b, h, t["k"].shape[-1], dv, generator=r, device=t["v"].device) if final_grad else None
    (o, f, g), (o2, f2, g2) = both(t, dout, dfinal, **kw)
    close(o, o2, TOL[dtype], "out")
    close(f, f2, STATE_TOL[dtype], "final_state")
    for n in g:
        assert g[n].dtype == t[n].dtype and g[n].shape == t[n].shape
        close(g[n], g2[n], STATE_TOL[dtype] if n == "initial_state" else TOL[dtype], "d" + n)


# ---- CPU: the reference's own form, and what is refused -------------------------------------------------------------
def test_ref_is_the_matrix_recurrence():
    t = {k: v.double() for k, v in inputs(1, 7, 1, 2, 3, 4, torch.float32, state=True, device="cpu").items()}
    out, final = gated_delta_rule_ref(**t, return_final_state=True, scale=0.5)
    for h in range(2):
        S = t["initial_state"][0, h]
        for i in range(7):
            k, q, a, b = t["k"][0, i, 0], t["q"][0, i, 0], t["g"][0, i, h].exp(), t["beta"][0, i, h]
            S = a * (torch.eye(3, dtype=S.dtype) - b * torch.outer(k, k)) @ S + b * torch.outer(k, t["v"][0, i, h])
            torch.testing.assert_close(out[0, i, h], 0.5 * q @ S)
        torch.testing.assert_close(final[0, h], S)


def test_ref_reverse_and_lengths_are_flips_and_cuts():
    t = inputs(2, 9, 1, 1, 4, 5, torch.float32, device="cpu")
    lens = torch.tensor([9, 4])
    out, final = gated_delta_rule_ref(**t, reverse=True, seq_lens=lens, return_final_state=True)
    for b, n in enumerate([9, 4]):
        cut = {k: v[b:b + 1, :n].flip(1) for k, v in t.items()}
        o, f = gated_delta_rule_ref(**cut, return_final_state=True)
        torch.testing.assert_close(out[b:b + 1, :n], o.flip(1))
        torch.testing.assert_close(final[b:b + 1], f)
        assert (out[b, n:] == 0).all()


@pytest.mark.parametrize("change, message", [
    (lambda t: {**t, "q": t["q"][..., :3]}, "expected"),
    (lambda t: {**t, "v": t["v"][:, :2]}, "batch and length"),
    (lambda t: {**t, "v": t["v"][:, :, :3], "g": t["g"][:, :, :3], "beta": t["beta"][:, :, :3]}, "multiple"),
    (lambda t: {**t, "g": t["g"][:, :, :1]}, "shape of v"),
    (lambda t: {**t, "k": t["k"].double()}, "one dtype"),
    (lambda t: {n: x.double() for n, x in t.items()}, "fp32, fp16 or bf16"),
    (lambda t: {**t, "beta": t["beta"].half()}, "g and beta"),
    (lambda t: {**t, "q": t["q"].repeat(1, 1, 1, 40), "k": t["k"].repeat(1, 1, 1, 40)}, "key heads"),
    (lambda t: t, "GPU"),
])
def test_refusals(change, message):
    t = inputs(1, 5, 2, 4, 4, 6, torch.float32, device="cpu")
    with pytest.raises(RuntimeError, match=message):
        gated_delta_rule_fn(**change(t))


def test_c_entry_refuses_without_a_gpu():
    """the C entries answer a bad block with a status and a message, before any launch"""
    import ctypes

    import vms_hip
    L = vms_hip.lib()
    P = vms_hip.GatedDeltaParams()
    assert L.vms_gated_delta_fwd(None, None) < 0 and L.vms_gated_delta_bwd(None, None) < 0
    assert L.vms_gated_delta_fwd(ctypes.byref(P), None) < 0 and b"empty" in L.vms_last_error()
    assert L.vms_gated_delta_workspace_bytes(ctypes.byref(P)) == 0
    P.batch = P.seqlen = P.heads = P.heads_k = 1
    P.dk, P.dv, P.dtype, P.gate_dtype = 16, 16, vms_hip.VMS_BF16, vms_hip.VMS_BF16
    P.q = P.k = P.v = P.g = P.beta = 256
    assert L.vms_gated_delta_fwd(ctypes.byref(P), None) < 0 and b"workspace" in L.vms_last_error()
    for field, value in (("dk", 129), ("dv", 0), ("dtype", 7), ("gate_dtype", vms_hip.VMS_F16), ("heads", 0), ("heads_k", 2)):
        keep = getattr(P, field)
        setattr(P, field, value)
        assert L.vms_gated_delta_fwd(ctypes.byref(P), None) < 0, field
        setattr(P, field, keep)
    n = L.vms_gated_delta_workspace_bytes(ctypes.byref(P))
    P.workspace, P.workspace_bytes = 256, n - 1
    assert L.vms_gated_delta_fwd(ctypes.byref(P), None) < 0 and b"too small" in L.vms_last_error()
    Q = vms_hip.GatedDeltaBwdParams()
    P.workspace_bytes = n
    Q.f = P
    assert L.vms_gated_delta_bwd(ctypes.byref(Q), None) < 0 and b"for_backward" in L.vms_last_error()


@pytest.mark.parametrize("dtype, for_backward, dv, most", [("VMS_BF16", 0, 32, 2**23), ("VMS_BF16", 1, 64, 2**22), ("VMS_F32", 0, 1, 2**23), ("VMS_F32", 1, 1, 2**22)])
def test_c_entry_refuses_launches_of_2_to_the_32_threads(dtype, for_backward, dv, most):
    """before any launch, and not one head earlier"""
    import ctypes

    import vms_hip
    L = vms_hip.lib()
    P = vms_hip.GatedDeltaParams()
    P.seqlen = P.heads_k = 1
    P.dk, P.dv, P.for_backward, P.q_seq_stride = 8, dv, for_backward, 2**40
    P.dtype = P.gate_dtype = getattr(vms_hip, dtype)
    P.q = P.k = P.v = P.g = P.beta = P.out = P.workspace = 256
    P.workspace_bytes = 2**62
    P.heads = 2048
    for batch, message in ((most // 2048, b"too large"), (most // 2048 - 1, b"strides")):   # (the next check, so that nothing is launched)
        P.batch = batch
        assert L.vms_gated_delta_fwd(ctypes.byref(P), None) < 0 and message in L.vms_last_error(), L.vms_last_error()


def test_c_messages_hold_their_condition():
    """conditions with a % in them used to be the format of the message"""
    import ctypes

    import vms_hip
    L = vms_hip.lib()
    P, S, N = vms_hip.GatedDeltaParams(), vms_hip.GatedDeltaStepParams(), vms_hip.SandwichNormParams()
    P.seqlen = P.batch = S.batch = 1
    P.heads = S.heads = 3
    P.heads_k = S.heads_k = 2
    for fn, p in ((L.vms_gated_delta_fwd, P), (L.vms_gated_delta_state_update, S)):
        assert fn(ctypes.byref(p), None) < 0
        assert L.vms_last_error() == b"vms check failed: p.heads % p.heads_k == 0 -- heads must be a multiple of heads_k"
    N.rows, N.cols, N.rows_per_gate = 4, 16, 3
    N.x = N.post_weight = N.pre_weight = N.gate = 256
    assert L.vms_sandwich_norm_fwd(ctypes.byref(N), None) < 0 and b"p.rows % p.rows_per_gate == 0 -- rows must" in L.vms_last_error()


def test_a_library_without_an_entry_is_refused_when_it_is_loaded(tmp_path, monkeypatch):
    """built before the entry was added, with the version of now: an ImportError that says what to do, not an AttributeError later"""
    import shutil
    import subprocess

    import vms_hip
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    (tmp_path / "old.c").write_text("\n".join(f"int {n}(void) {{ return {vms_hip.ABI_VERSION}; }}" for n in vms_hip.EXPORTS if "gated_delta" not in n))
    subprocess.check_call([cc, "-shared", "-fPIC", "-o", str(tmp_path / "old.so"), str(tmp_path / "old.c")])
    monkeypatch.setattr(vms_hip, "LIB_PATH", str(tmp_path / "old.so"))
    monkeypatch.setattr(vms_hip, "_lib", None)
    with pytest.raises(ImportError, match="vms_gated_delta_fwd.*rebuild"):
        vms_hip.lib()


def test_sizes_beyond_32_bits_are_refused():
    """a length of 2^32 + 3 must not be taken for one of 3"""
    t = inputs(1, 1, 1, 1, 4, 6, torch.float32, device="cpu")
    big = {k: v.expand(1, 2**32 + 3, *v.shape[2:]) for k, v in t.items()}
    with pytest.raises(RuntimeError, match="2\\^31"):
        gated_delta_rule_fn(**big)


# ---- GPU ------------------------------------------------------------------------------------------------------------
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("l", [1, 2, 17, 63, 64, 65, 130, 197])
def test_lengths(l, dtype):
    compare(inputs(2, l, 2, 2, 64, 64, dtype, state=True, seed=l))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reverse", [False, True])
def test_first_gate_without_a_state(reverse, dtype):
    """a gate with nothing to forget has gradient 0, not two terms' roundings; with a state it has one"""
    for l in (1, 70):
        for state in (False, True):
            leaf = {k: v.requires_grad_() for k, v in inputs(2, l, 1, 2, 32, 32, dtype, state=state, seed=l).items()}
            dg, = torch.autograd.grad(gated_delta_rule_fn(**leaf, reverse=reverse).float().square().sum(), leaf["g"])
            assert ((dg[:, l - 1 if reverse else 0] == 0) != state).all() and (l == 1 or (dg[:, 1:-1] != 0).any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dk, dv", [(1, 1), (3, 5), (8, 130), (40, 72), (65, 33), (100, 100), (128, 128), (128, 17), (16, 272)])
def test_head_sizes(dk, dv, dtype):
    compare(inputs(1, 90, 1, 2, dk, dv, dtype, state=True, seed=dk + dv))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hk, h, b", [(1, 1, 1), (1, 5, 1), (2, 4, 3), (3, 9, 2), (8, 8, 2)])
def test_shared_heads(hk, h, b, dtype):
    compare(inputs(b, 70, hk, h, 32, 48, dtype, seed=h))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dk, dv", [(40, 72), (64, 64), (50, 70), (100, 96), (104, 90), (128, 128)])
def test_many_heads(dk, dv, dtype):
    """enough heads for workgroups of 32 columns, the last one partly outside; lengths of one to four chunks"""
    lens = torch.tensor([200, 1, 129, 64, 63], dtype=torch.int32, device="cuda")
    compare(inputs(5, 200, 8, 16, dk, dv, dtype, state=True, seed=dk), seq_lens=lens, reverse=dk % 8 == 0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reverse", [False, True])
def test_ragged(reverse, dtype):
    """lengths: none, one, inside a chunk, whole, beyond (clamped), negative (clamped); what stands in the padding is never read"""
    t = inputs(6, 140, 2, 2, 64, 40, dtype, state=True, seed=3)
    lens = torch.tensor([0, 1, 77, 140, 999, -5], dtype=torch.int32, device="cuda")
    for b, n in enumerate([0, 1, 77, 140, 140, 0]):
        for k in ("q", "k", "v", "g", "beta"):
            t[k][b, n:] = float("nan")
    r = torch.Generator(device="cuda").manual_seed(5)
    dout = torch.randn(t["v"].shape, generator=r, device="cuda").to(dtype)
    dfinal = torch.randn(6, 2, 64, 40, generator=r, device="cuda")
    (o, f, g), (o2, f2, g2) = both(t, dout, dfinal, reverse=reverse, seq_lens=lens)
    close(o, o2, TOL[dtype], "out")
    close(f, f2, STATE_TOL[dtype], "final_state")
    for n in g:
        assert not g[n].isnan().any(), n
        close(g[n], g2[n].nan_to_num(), STATE_TOL[dtype] if n == "initial_state" else TOL[dtype], "d" + n)
    for b, n in enumerate([0, 1, 77, 140, 140, 0]):
        assert (o[b, n:] == 0).all() and all((g[k][b, n:] == 0).all() for k in ("q", "k", "v", "g", "beta"))
    assert torch.equal(f[0], t["initial_state"][0]) and torch.equal(g["initial_state"][0], dfinal[0])


@pytest.mark.gpu
def test_int64_lengths_do_not_wrap():
    t = inputs(2, 20, 1, 1, 16, 16, torch.float32)
    a = gated_delta_rule_fn(**t, seq_lens=torch.tensor([2**32 + 3, 7], device="cuda"))
    b = gated_delta_rule_fn(**t, seq_lens=torch.tensor([20, 7], dtype=torch.int32, device="cuda"))
    assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("reverse", [False, True])
def test_reverse_is_the_flipped_walk(reverse):
    t = inputs(2, 133, 1, 2, 64, 64, torch.bfloat16, state=True)
    flipped = {k: v if k == "initial_state" else v.flip(1) for k, v in t.items()}
    a, sa = gated_delta_rule_fn(**t, reverse=reverse, return_final_state=True)
    b, sb = gated_delta_rule_fn(**flipped, reverse=not reverse, return_final_state=True)
    assert torch.equal(a, b.flip(1)) and torch.equal(sa, sb)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(dtype):
    """views of one fused projection, heads before tokens, rows at odd offsets, an expanded batch, a strided last axis"""
    t = inputs(2, 100, 2, 2, 40, 56, dtype)
    want = gated_delta_rule_fn(**t)
    fused = torch.cat([t["q"].flatten(2), t["k"].flatten(2), t["v"].flatten(2), t["v"].new_zeros(2, 100, 3)], -1)
    q, k, v, _ = fused.split([80, 80, 112, 3], -1)
    assert torch.equal(want, gated_delta_rule_fn(q.unflatten(-1, (2, 40)), k.unflatten(-1, (2, 40)), v.unflatten(-1, (2, 56)), t["g"], t["beta"]))
    heads_first = {n: x.transpose(1, 2).contiguous().transpose(1, 2) for n, x in t.items()}
    assert torch.equal(want, gated_delta_rule_fn(**heads_first))
    odd = {}
    for n, x in t.items():
        buf = torch.empty(x.numel() + 1, dtype=dtype, device="cuda")
        odd[n] = buf[1:].view(x.shape).copy_(x)
    assert torch.equal(want, gated_delta_rule_fn(**odd))
    strided = {n: torch.stack([x, x], -1)[..., 0] for n, x in t.items()}
    assert torch.equal(want, gated_delta_rule_fn(**strided))
    one = {n: x[:1] for n, x in t.items()}
    wide = {n: x[:1].expand(3, *x.shape[1:]) for n, x in t.items()}
    assert torch.equal(gated_delta_rule_fn(**one).expand(3, -1, -1, -1), gated_delta_rule_fn(**wide))
    leaf = {n: x[:1].detach().clone().requires_grad_() for n, x in t.items()}
    gated_delta_rule_fn(**{n: x.expand(3, *x.shape[1:]) for n, x in leaf.items()}).sum().backward()   # an expanded gradient too
    compare({n: x.detach() for n, x in leaf.items()}, final_grad=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hk, dk, dv", [(2, 40, 56), (1, 64, 64), (2, 33, 17)])
def test_gradients_of_strided_calls(hk, dk, dv, dtype):
    """slices of one projection, heads before tokens, a strided last axis and a gradient laid out otherwise: the bits of the contiguous call"""
    t = inputs(2, 100, hk, 2, dk, dv, dtype, seed=dk)
    dout = torch.randn(t["v"].shape, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda").to(dtype)

    def run(make, dout):
        leaf = {n: make(x).detach().requires_grad_() for n, x in t.items()}
        return torch.autograd.grad(gated_delta_rule_fn(**leaf), list(leaf.values()), dout)
    want = run(lambda x: x, dout)
    heads_first = lambda x: x.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
    tokens_first = lambda x: x.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    strided = lambda x: torch.stack([x, x], -1)[..., 0]  # noqa: E731
    slices = lambda x: torch.cat([x[..., :1], x, x], -1)[..., 1:x.shape[-1] + 1]  # noqa: E731
    for turn in (heads_first, tokens_first, strided, slices):
        for d in (dout, turn(dout)):
            assert turn(dout).stride() != dout.stride()
            for n, a, b in zip(t, run(turn, d), want):
                assert torch.equal(a, b), (turn, n)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients_of_expanded_leaves(dtype):
    """one batch entry seen three times, an expanded gradient: the leaves get the sum of three equal gradients.  autograd adds them in the leaf's type: two more
    roundings of up to three times the size"""
    t = inputs(1, 100, 2, 2, 40, 56, dtype)
    leaf = {n: x.clone().requires_grad_() for n, x in t.items()}
    gated_delta_rule_fn(**{n: x.expand(3, *x.shape[1:]) for n, x in leaf.items()}).sum().backward()
    wide = {n: x.double().requires_grad_() for n, x in t.items()}
    gated_delta_rule_ref(**{n: x.expand(3, *x.shape[1:]) for n, x in wide.items()}).sum().backward()
    for n in t:
        close(leaf[n].grad, wide[n].grad, TOL[dtype] + 2 * torch.finfo(dtype).eps / 2, "d" + n)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_fp32_gates(dtype):
    compare(inputs(2, 150, 1, 2, 64, 64, dtype, gate_dtype=torch.float32))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gate", [-math.inf, -300.0, -30.0, 0.0])
def test_strong_and_absent_decay(gate, dtype):
    """a state that is forgotten whole (also several times in a chunk), hardly, or never; beta 0 and 1"""
    t = inputs(1, 200, 1, 2, 32, 32, dtype, state=True)
    t["g"][:, ::7] = gate
    t["beta"][:, ::5] = 0
    t["beta"][:, 1::5] = 1
    r = torch.Generator(device="cuda").manual_seed(1)
    dout = torch.randn(t["v"].shape, generator=r, device="cuda").to(dtype)
    (o, f, g), (o2, f2, g2) = both(t, dout, None)
    close(o, o2, TOL[dtype], "out")
    close(f, f2, STATE_TOL[dtype], "final_state")
    for n in g:
        want = g2[n].nan_to_num(0.0) if n == "g" else g2[n]   # autograd of exp(-inf) * 0 may be NaN; the gradient is 0 there
        close(g[n], want, STATE_TOL[dtype] if n == "initial_state" else TOL[dtype], "d" + n)


@pytest.mark.gpu
def test_equal_keys():
    """every key the same and beta 1: the triangular inverse is a difference of neighbours; a series in powers would lose it.
    The state is replaced whole at every token, so that dg is 0: a sum of up to 3 x 64 terms (q.dq, k.dk as left and right factor) that
    cancel.  Each term is an fp32 sum of 16 products of values that passed at most four fp32 sums of up to 64, i.e. off by less than
    (16 + 4 * 64) 2^-24 = 1.6e-5 of its size, so dg is held to 2e-5 of the largest term, not of itself."""
    t = inputs(1, 128, 1, 1, 16, 16, torch.float32)
    t["k"] = t["k"][:, :1].expand(-1, 128, -1, -1).contiguous()
    t["g"] = t["g"] * 0
    t["beta"] = t["beta"] * 0 + 1
    dout = torch.randn(t["v"].shape, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    (o, f, g), (o2, f2, g2) = both(t, dout)
    close(o, o2, 2e-5)
    close(f, f2, 2e-5)
    for n in ("q", "k", "v", "beta"):
        close(g[n], g2[n], 2e-5, "d" + n)
    term = max((t[n].double() * g2[n]).sum(-1).abs().max().item() for n in ("q", "k"))
    assert (g["g"] - g2["g"]).abs().max().item() <= 2e-5 * term


@pytest.mark.gpu
def test_differences():
    """directional differences of the fp32 kernels: f is computed to ~1e-7 of its scale (~60), h = 3e-3: rounding 6e-6 / 2 h = 1e-3, truncation
    of the order of (h sqrt(24))^2 = 2e-4 of the gradient per factor k of a product over few tokens that still matter"""
    t = inputs(1, 75, 1, 2, 24, 24, torch.float32, state=True)
    r = torch.Generator(device="cuda").manual_seed(9)
    dout = torch.randn(t["v"].shape, generator=r, device="cuda")

    def f(x):
        return (gated_delta_rule_fn(**x).double() * dout.double()).sum()

    leaf = {k: v.clone().requires_grad_() for k, v in t.items()}
    grads = dict(zip(leaf, torch.autograd.grad(f(leaf), list(leaf.values()))))
    for n in t:
        d = torch.randn(t[n].shape, generator=r, device="cuda")
        h = 3e-3
        up, down = ({**t, n: t[n] + s * h * d} for s in (1, -1))
        diff = ((f(up) - f(down)) / (2 * h)).item()
        got = (grads[n].double() * d).sum().item()
        size = (grads[n].double().norm() * d.double().norm()).item() / math.sqrt(d.numel())
        assert abs(diff - got) <= 2e-2 * size + 5e-3, (n, diff, got, size)


@pytest.mark.gpu
def test_same_call_same_bits():
    t = inputs(2, 300, 2, 4, 64, 64, torch.bfloat16, state=True)
    runs = []
    for _ in range(2):
        leaf = {k: v.clone().requires_grad_() for k, v in t.items()}
        out, s = gated_delta_rule_fn(**leaf, return_final_state=True)
        runs.append([out, s, *torch.autograd.grad((out.float().sum() + s.sum()), list(leaf.values()))])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


@pytest.mark.gpu
def test_inference_equals_training_forward():
    t = inputs(2, 100, 1, 2, 64, 96, torch.bfloat16)
    a = gated_delta_rule_fn(**t)
    b = gated_delta_rule_fn(**{k: v.clone().requires_grad_() for k, v in t.items()})
    assert torch.equal(a, b)


@pytest.mark.gpu
def test_state_carries_over():
    """a sequence in two calls, state handed on, equals one call at the rounding of the outputs"""
    t = inputs(1, 192, 1, 2, 64, 64, torch.float32)
    whole, s = gated_delta_rule_fn(**t, return_final_state=True)
    a, sa = gated_delta_rule_fn(**{k: v[:, :100] for k, v in t.items()}, return_final_state=True)
    b, sb = gated_delta_rule_fn(**{k: v[:, 100:] for k, v in t.items()}, initial_state=sa, return_final_state=True)
    close(torch.cat([a, b], 1), whole, 2e-5)
    close(sb, s, 2e-5)


@pytest.mark.gpu
def test_nothing_to_walk_over():
    t = inputs(2, 0, 1, 2, 8, 8, torch.float32, state=True)
    out, s = gated_delta_rule_fn(**t, return_final_state=True)
    assert out.shape == (2, 0, 2, 8) and torch.equal(s, t["initial_state"])
    t = inputs(0, 4, 1, 2, 8, 8, torch.float32)
    out, s = gated_delta_rule_fn(**t, return_final_state=True)
    assert out.shape == (0, 4, 2, 8) and s.shape == (0, 2, 8, 8)


@pytest.mark.gpu
@pytest.mark.parametrize("b, l, h", [(2, 0, 2), (0, 4, 2), (2, 4, 0)])
def test_gradients_of_nothing(b, l, h):
    """no token, no batch entry, no head: zeros of every leaf's shape, and the state's own gradient passes through"""
    for state in (False, True):
        leaf = {k: v.requires_grad_() for k, v in inputs(b, l, 2, h, 8, 8, torch.bfloat16, state=state).items()}
        out, s = gated_delta_rule_fn(**leaf, return_final_state=True)
        assert out.shape == (b, l, h, 8) and out.dtype == torch.bfloat16 and s.shape == (b, h, 8, 8) and s.dtype == torch.float32
        for heads in ((out, s), (out,), (s,)):
            grads = torch.autograd.grad(heads, list(leaf.values()), [torch.ones_like(x) for x in heads], retain_graph=True)
            for n, g in zip(leaf, grads):
                want = 1 if n == "initial_state" and any(x is s for x in heads) else 0
                assert g.shape == leaf[n].shape and (g == want).all(), n
    if l == 0:   # whatever the state holds
        t = inputs(b, l, 2, h, 8, 8, torch.bfloat16, state=True)
        t["initial_state"][0] = float("nan")
        t["initial_state"][1] = float("inf")
        assert torch.equal(gated_delta_rule_fn(**t, return_final_state=True)[1].nan_to_num(5.0), t["initial_state"].nan_to_num(5.0))


@pytest.mark.gpu
def test_only_some_gradients():
    """a gradient that arrives through the final state alone; leaves that want none"""
    t = inputs(1, 70, 1, 1, 16, 16, torch.float32)
    v = t["v"].clone().requires_grad_()
    _, s = gated_delta_rule_fn(t["q"], t["k"], v, t["g"], t["beta"], return_final_state=True)
    got, = torch.autograd.grad(s.square().sum(), v)
    v2 = t["v"].double().requires_grad_()
    _, s2 = gated_delta_rule_ref(*(t[n].double() for n in "qk"), v2, t["g"].double(), t["beta"].double(), return_final_state=True)
    close(got, torch.autograd.grad(s2.square().sum(), v2)[0], 4e-5)


@pytest.mark.gpu
def test_on_another_stream_and_captured():
    t = inputs(2, 150, 1, 2, 64, 64, torch.bfloat16)
    want, ws = gated_delta_rule_fn(**t, return_final_state=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, gs = gated_delta_rule_fn(**t, return_final_state=True)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(want, got) and torch.equal(ws, gs)

    leaf = {k: v.clone().requires_grad_() for k, v in t.items()}
    dout = torch.randn_like(want)
    eager = torch.autograd.grad(gated_delta_rule_fn(**leaf), list(leaf.values()), dout)
    static = {k: v.clone().requires_grad_() for k, v in t.items()}
    with torch.cuda.stream(side):
        torch.autograd.grad(gated_delta_rule_fn(**static), list(static.values()), dout)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = gated_delta_rule_fn(**static)
        grads = torch.autograd.grad(out, list(static.values()), dout)
    for k in range(3):
        with torch.no_grad():
            for n in static:
                static[n].copy_(t[n] if k != 1 else t[n] * 0.5)
        graph.replay()
        torch.cuda.synchronize()
        if k != 1:
            assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(grads, eager))
        else:
            half = {n: (x * 0.5).requires_grad_() for n, x in t.items()}
            o = gated_delta_rule_fn(**half)
            assert torch.equal(out, o)
            assert all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(o, list(half.values()), dout)))


@pytest.mark.gpu
def test_two_calls_at_once():
    """two streams, two host threads: every call has its own workspace"""
    import threading
    sets = [inputs(2, 300, 2, 4, 64, 64, torch.bfloat16, seed=i) for i in range(2)]
    douts = [torch.randn_like(t["v"]) for t in sets]

    def run(i):
        leaf = {k: v.clone().requires_grad_() for k, v in sets[i].items()}
        out = gated_delta_rule_fn(**leaf)
        return [out.detach(), *torch.autograd.grad(out, list(leaf.values()), douts[i])]
    want = [run(i) for i in range(2)]
    torch.cuda.synchronize()
    got = [[], []]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                got[i].append(run(i))
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(2):
        assert len(got[i]) == 5 and all(torch.equal(a, b) for g in got[i] for a, b in zip(g, want[i]))


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    t = inputs(2, 70, 1, 1, 32, 32, torch.bfloat16)
    far = dict(t)
    for k in ("q", "k", "v"):
        room = torch.empty(2**31 + 8 + 70 * 32, dtype=torch.bfloat16, device="cuda")
        far[k] = room.as_strided((2, 70, 1, 32), (2**31 + 8, 32, 32, 1))
        far[k].copy_(t[k])
    res = []
    for x in (t, far):
        leaf = {k: v.detach().requires_grad_() for k, v in x.items()}
        out = gated_delta_rule_fn(**leaf)
        res.append([out, *torch.autograd.grad(out, list(leaf.values()), torch.ones_like(out))])
    assert all(torch.equal(a, b) for a, b in zip(*res))


@pytest.mark.gpu
def test_backward_twice_and_one_tensor_for_two():
    t = inputs(2, 130, 2, 2, 32, 32, torch.bfloat16)
    leaf = {k: v.clone().requires_grad_() for k, v in t.items()}
    out = gated_delta_rule_fn(**leaf)
    dout = torch.randn_like(out)
    a = torch.autograd.grad(out, list(leaf.values()), dout, retain_graph=True)
    b = torch.autograd.grad(out, list(leaf.values()), dout)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    x = t["k"].clone().requires_grad_()   # q, k and v one tensor: the gradients add up
    parts = [t["k"].clone().requires_grad_() for _ in range(3)]
    one, = torch.autograd.grad(gated_delta_rule_fn(x, x, x, t["g"], t["beta"]), x, dout)
    three = torch.autograd.grad(gated_delta_rule_fn(*parts, t["g"], t["beta"]), parts, dout)
    # autograd adds the three in bf16, in some order: one rounding (2^-8) of a sum of two, one of the whole
    a, b, c = (p.double() for p in three)
    two = max(x.abs().max().item() for x in (a + b, a + c, b + c))
    top = (a + b + c).abs().max().item()
    close(one, a + b + c, 2**-8 * (two + 2**-8 * two + top) / top, "dx")


@pytest.mark.gpu
def test_a_nan_stays_behind_its_chunk():
    t = inputs(1, 200, 1, 1, 32, 32, torch.bfloat16)
    want = gated_delta_rule_fn(**t)
    t["v"][0, 130] = float("nan")
    got = gated_delta_rule_fn(**t)
    assert torch.equal(got[0, :128], want[0, :128]) and got[0, 130:].isnan().all()


@pytest.mark.gpu
def test_sizes_beyond_32_bits_are_refused_by_the_compiled_call():
    t = inputs(1, 1, 1, 1, 4, 6, torch.float32)
    with pytest.raises(RuntimeError, match="2\\^31"):
        gated_delta_rule_fn(**{k: v.expand(1, 2**32 + 3, *v.shape[2:]) for k, v in t.items()})


@pytest.mark.gpu
def test_compiled_and_ctypes_calls_are_one(monkeypatch):
    """the compiled binding's node and the ctypes one: the same bits, the same refusals, and no second derivative in either"""
    import vms_hip
    ext = vms_hip.ext()
    assert ext is not None
    t = inputs(2, 100, 1, 2, 40, 48, torch.bfloat16, state=True)
    lens = torch.tensor([100, 31], device="cuda")
    dout = torch.randn_like(t["v"])
    runs = []
    for use in (ext, None):
        monkeypatch.setattr(vms_hip, "_ext", use)
        leaf = {k: v.clone().requires_grad_() for k, v in t.items()}
        out, s = gated_delta_rule_fn(**leaf, return_final_state=True, reverse=True, seq_lens=lens)
        runs.append([out, s, *torch.autograd.grad((out, s), list(leaf.values()), (dout, s.detach()))])
        with torch.no_grad():
            runs[-1].append(gated_delta_rule_fn(**leaf, scale=0.5))
        leaf = {k: v.float().requires_grad_() for k, v in t.items()}
        g, = torch.autograd.grad(gated_delta_rule_fn(**leaf).square().sum(), leaf["v"], create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.sum().backward()
        for bad in ({"q": t["q"][..., :3]}, {"k": t["k"].float()}, {"beta": t["beta"].half()}, {"initial_state": t["initial_state"].half()},
                    {"seq_lens": lens.float()}, {"seq_lens": lens[:1]}, {"g": t["g"].cpu()}):
            with pytest.raises(RuntimeError, match="gated_delta_rule"):
                gated_delta_rule_fn(**{**t, **bad})
    assert all(torch.equal(a, b) for a, b in zip(*runs))
