"""Gated delta rule where its sums cancel: keys and queries that share a direction, beta near 1, slow decay; gates in fp32 beside 16-bit q, k, v;
sequences of many chunks.

Tolerances, fixed before the first run.  An operand of the kernels' products is off by at most 2^-16 of itself for 16-bit inputs (two bf16 planes), 2^-24
for fp32, where sums of up to 64 + 128 terms add sqrt(192) 2^-24.  Correlated keys make outputs and gradients differences of larger terms:
up to 64 times larger is allowed for, so that what is compared is off in the norm by at most
  16-bit results:                    eps / 2 of their own rounding + 64 * 2^-16
  fp32 results of 16-bit inputs:     64 * 2^-16
  fp32:                              64 * sqrt(192) * 2^-24
dg alone cancels further: dg_t is the sum, over the tokens from t to the end of its 64, of q.dq - du.(v - e) - du.e (du = the gradient of u, e = what v leaves of the
state's guess; each of the three a product of two computed vectors, each of those off by 3 * 2^-16 of itself: two residuals, one product of residuals left out), and with equal
keys the three nearly cancel.  6 * 2^-16 of every term, times sqrt(64) for a sum of up to 64 errors: 48 * 2^-16 of the three terms' norm, which is up to 18 times dg's here.
Independent keys: the tolerances of test_gated_delta; the fp32 gradients of fp32 gates pass at most eight products in a row (state to state four, then U or Y, Z, W or X,
the row's sum), each off by at most 3 * 2^-16: 24 * 2^-16 of the largest."""
import math

import pytest
import torch

from mamba_ssm.ops.gated_delta_rule import gated_delta_rule_fn, gated_delta_rule_ref
from test_gated_delta import DTYPES, TOL, both, close, compare, inputs

PLANES = {torch.float32: math.sqrt(192) * 2**-24, torch.float16: 2**-16, torch.bfloat16: 2**-16}


def norm_close(got, want, dtype, what, terms=None):
    half = 0 if got.dtype == torch.float32 else torch.finfo(got.dtype).eps / 2
    off, size = (got.double() - want).norm().item(), want.norm().item()
    tol = half * size + (64 * PLANES[dtype] * size if terms is None else 48 * PLANES[dtype] * terms)
    assert off <= tol, f"{what}: off by {off / size:.2e} of its norm > {tol / size:.2e}"


def gate_terms(t, grads):
    """norm of the three terms that dg is a sum of; heads of q and k are those of v here or shared by all"""
    u = {n: x.double() for n, x in t.items()}
    rep = u["v"].shape[2] // u["k"].shape[2]
    k = u["k"].repeat_interleave(rep, 2)
    S, guess = u["initial_state"], []
    for i in range(k.shape[1]):
        S = S * u["g"][:, i].exp()[..., None, None]
        guess.append((S * k[:, i, :, :, None]).sum(-2))
        S = S + k[:, i, :, :, None] * (u["beta"][:, i, :, None] * (u["v"][:, i] - guess[-1]))[..., None, :]
    guess = torch.stack(guess, 1)
    # (shared heads: dq is a sum over them, whose size stands for each one's; dv = beta du)
    parts = [(u["q"] * grads["q"]).sum(-1).repeat_interleave(rep, 2), (grads["v"] * guess).sum(-1), (grads["v"] * (u["v"] - guess)).sum(-1)]
    return torch.stack(parts).norm().item()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, gate_dtype", [(torch.float32, torch.float32), (torch.float16, torch.float16), (torch.float16, torch.float32),
                                               (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("hk, d, cos, beta, decay", [(2, 64, 0.9, 0.95, 0.02), (1, 64, 0.99, 1.0, 0.02), (2, 128, 0.9, 0.98, 0.002), (1, 128, 0.99, 1.0, 0.002)])
def test_correlated_keys(hk, d, cos, beta, decay, dtype, gate_dtype):
    l, h = 512, 2
    t = inputs(1, l, hk, h, d, d, torch.float32, state=True, seed=d)
    r = torch.Generator(device="cuda").manual_seed(1)
    common = torch.randn(hk, d, generator=r, device="cuda")
    common /= common.norm(dim=-1, keepdim=True)
    for n in ("q", "k"):
        x = math.sqrt(1 - cos) * t[n] + math.sqrt(cos) * common
        t[n] = (x / x.norm(dim=-1, keepdim=True)).to(dtype)
    t["v"] = t["v"].to(dtype)
    t["g"] = (-decay * torch.rand(1, l, h, generator=r, device="cuda")).to(gate_dtype)
    t["beta"] = torch.full_like(t["g"], beta)
    dout = torch.randn(t["v"].shape, generator=r, device="cuda").to(dtype)
    (o, f, g), (o2, f2, g2) = both(t, dout)
    norm_close(o, o2, dtype, "out")
    norm_close(f, f2, dtype, "final_state")
    for n in g:
        norm_close(g[n], g2[n], dtype, "d" + n, gate_terms(t, g2) if n == "g" else None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dk, dv", [(64, 64), (128, 128), (40, 70)])
def test_gradients_of_fp32_gates(dk, dv, dtype):
    """they are fp32, and as good as the operands' 16 bits: not as a 16-bit result's"""
    t = inputs(2, 200, 1, 2, dk, dv, dtype, state=True, gate_dtype=torch.float32, seed=dk)
    dout = torch.randn(t["v"].shape, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").to(dtype)
    (_, _, g), (_, _, g2) = both(t, dout)
    for n in ("g", "beta"):
        close(g[n], g2[n], 24 * 2**-16, "d" + n)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("l, reverse", [(2304, False), (4101, True)])
def test_many_chunks(l, reverse, dtype):
    """36 and 65 chunks of a state that hardly decays: nothing grows along the walk"""
    t = inputs(1, l, 1, 2, 64, 48, dtype, state=True, seed=l)
    t["g"] = t["g"] * 0.01
    compare(t, reverse=reverse)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("b, l, hk, h, dk, dv", [(1, 200, 2, 2, 64, 64), (1, 300, 1, 2, 128, 128), (2, 130, 1, 1, 40, 72), (1, 150, 2, 2, 100, 33), (40, 70, 4, 4, 64, 32),
                                                 (20, 129, 8, 8, 128, 128), (20, 66, 4, 8, 96, 100), (70, 65, 2, 2, 50, 50)])
def test_fp32_states_of_16_bit_inputs(b, l, hk, h, dk, dv, dtype):
    """calls with a state in or out carry what they compute to 2^-24: the state, its gradient and those of fp32 gates are off, in the norm, by what fp32 sums leave.
    A rounding is 2^-24 / sqrt(3) on average: sqrt(64 + 128) of them in a row of sums, four products in a row, each with three residuals of that size:
    (sqrt(192) + 4 * 3) 2^-24 / sqrt(3) = 9e-7; twice that for what the matrix cores' order of adding costs.  (Two planes leave 4e-6.)"""
    t = inputs(b, l, hk, h, dk, dv, dtype, state=True, gate_dtype=torch.float32, seed=dk + dv)
    r = torch.Generator(device="cuda").manual_seed(3)
    dout = torch.randn(t["v"].shape, generator=r, device="cuda").to(dtype)
    dfinal = 0.3 * torch.randn(b, h, dk, dv, generator=r, device="cuda")
    (o, f, g), (o2, f2, g2) = both(t, dout, dfinal, reverse=b > 1)
    for n, got, want in (("final", f, f2), *((n, g[n], g2[n]) for n in ("initial_state", "g", "beta"))):
        off = ((got.double() - want).norm() / want.norm()).item()
        assert got.dtype == torch.float32 and off <= 1.8e-6, (n, off)
    with torch.no_grad():
        for kw in ({}, {"initial_state": t["initial_state"]}):
            x = {n: v for n, v in t.items() if n != "initial_state"} | kw
            _, got = gated_delta_rule_fn(**x, return_final_state=True, reverse=b > 1)
            _, want = gated_delta_rule_ref(**{n: v.double() for n, v in x.items()}, return_final_state=True, reverse=b > 1)
            assert ((got.double() - want).norm() / want.norm()).item() <= 1.8e-6


def stateless(t, dout, **kw):
    """(out, gradients) of the kernels and in 64 bits, no state in or out: 16-bit inputs are carried in two planes"""
    res = []
    for fn, cast in ((gated_delta_rule_fn, lambda x: x.detach().clone()), (gated_delta_rule_ref, lambda x: x.detach().double())):
        leaf = {k: cast(v).requires_grad_() for k, v in t.items()}
        out = fn(**leaf, **kw)
        res.append((out, dict(zip(leaf, torch.autograd.grad(out, list(leaf.values()), dout.to(out.dtype))))))
    return res


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, gate_dtype", [(torch.float32, torch.float32), (torch.float16, torch.float32), (torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("hk, d, cos, beta, decay", [(2, 64, 0.9, 0.95, 0.02), (1, 64, 0.99, 1.0, 0.02), (1, 128, 0.99, 1.0, 0.002)])
def test_correlated_keys_without_states(hk, d, cos, beta, decay, dtype, gate_dtype):
    l, h = 512, 2
    t = inputs(1, l, hk, h, d, d, torch.float32, seed=d + 1)
    r = torch.Generator(device="cuda").manual_seed(2)
    common = torch.randn(hk, d, generator=r, device="cuda")
    common /= common.norm(dim=-1, keepdim=True)
    for n in ("q", "k"):
        x = math.sqrt(1 - cos) * t[n] + math.sqrt(cos) * common
        t[n] = (x / x.norm(dim=-1, keepdim=True)).to(dtype)
    t["v"] = t["v"].to(dtype)
    t["g"] = (-decay * torch.rand(1, l, h, generator=r, device="cuda")).to(gate_dtype)
    t["beta"] = torch.full_like(t["g"], beta)
    dout = torch.randn(t["v"].shape, generator=r, device="cuda").to(dtype)
    (o, g), (o2, g2) = stateless(t, dout)
    norm_close(o, o2, dtype, "out")
    for n in g:
        norm_close(g[n], g2[n], dtype, "d" + n, gate_terms({**t, "initial_state": torch.zeros(1, h, d, d, device="cuda")}, g2) if n == "g" else None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b, l, hk, h, dk, dv", [(2, 1, 2, 2, 64, 64), (1, 150, 2, 2, 100, 33), (1, 150, 2, 2, 96, 40), (2, 200, 1, 3, 128, 128), (1, 130, 2, 2, 50, 70),
                                                 (2, 77, 1, 2, 100, 50), (20, 129, 8, 8, 128, 128), (40, 70, 4, 4, 64, 32), (20, 66, 4, 8, 96, 100), (70, 65, 2, 2, 50, 50)])
def test_training_without_states(b, l, hk, h, dk, dv, dtype):
    """every form of the kernels that keeps two planes (few and many heads, 64 and 128 wide, whole and odd sizes, shared heads), ragged, both directions"""
    t = inputs(b, l, hk, h, dk, dv, dtype, gate_dtype=torch.float32, seed=dk + dv)
    r = torch.Generator(device="cuda").manual_seed(4)
    dout = torch.randn(t["v"].shape, generator=r, device="cuda").to(dtype)
    lens = torch.randint(0, l + 1, (b,), generator=r, device="cuda") if b > 2 else None
    (o, g), (o2, g2) = stateless(t, dout, reverse=b > 1, seq_lens=lens)
    close(o, o2, TOL[dtype], "out")
    for n in g:
        close(g[n], g2[n], TOL[dtype] if dtype == torch.float32 or n in "qkv" else 24 * 2**-16, "d" + n)
    again = stateless(t, dout, reverse=b > 1, seq_lens=lens)[0]
    assert torch.equal(again[0], o) and all(torch.equal(again[1][n], g[n]) for n in g)
