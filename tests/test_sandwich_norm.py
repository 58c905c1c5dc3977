"""sandwich_norm_fn (norm after a block, gate, scaled residual add, norm before the next) against its formula in 64 bits.

Tolerances, relative to the largest value compared: the arithmetic is fp32 over rows of up to 8192 (sums by lane, wave and team, i.e. chains of
under 64 additions: 64 * 2^-24 = 4e-6 per statistic, two statistics and their gradients in a row: 2e-5); sums over rows chain up to
rows / 1024 + 80 additions, under 256 here: 2e-5 as well; one rounding to a 16-bit result: 2^-8 bf16, 2^-11 fp16."""
import os

import pytest
import torch

from mamba_ssm.ops.gated_delta_rule import gated_delta_rule_fn
from mamba_ssm.ops.triton.layernorm import layer_norm_fn, rms_norm_fn, sandwich_norm_fn, sandwich_norm_ref
from test_gated_delta import DTYPES, close, inputs

TOL = {torch.float32: 2e-5, torch.float16: 2e-5 + 2**-11, torch.bfloat16: 2e-5 + 2**-8}


def make(shape, dtype, res_dtype=None, bias=True, gate="none", gate_dtype=torch.float32, weight_dtype=torch.float32, seed=0, device="cuda"):
    r = torch.Generator(device=device).manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=r, device=device)  # noqa: E731
    n = shape[-1]
    t = {"x": (randn(*shape) + 0.5).to(dtype), "residual": None if res_dtype is None else (2 * randn(*shape)).to(res_dtype),
         "post_weight": (1 + 0.2 * randn(n)).to(weight_dtype), "pre_weight": (1 + 0.2 * randn(n)).to(weight_dtype)}
    if bias:
        t |= {"post_bias": (0.1 * randn(n)).to(weight_dtype), "pre_bias": (0.1 * randn(n)).to(weight_dtype)}
    gates = {"channel": (n,), "ones": (1,) * (len(shape) - 1) + (n,), "batch": (shape[0],) + (1,) * (len(shape) - 2) + (n,), "token": shape}
    if gate != "none":
        t["gate"] = (0.5 + 0.3 * randn(*gates[gate])).to(gate_dtype)
    return t


def compare(t, tol_scale=1.0, dx_cancels=False, **kw):
    """dx_cancels: dx = rstd (s - xhat mean(s xhat) - mean(s)), s = gate dr post_weight, is a difference of terms of the size rstd |s|, each computed
    to TOL of itself; where they cancel (layer norm of two values: xhat = +-1 whatever x is, dx = eps / variance of them) dx is held to TOL of the terms"""
    r = torch.Generator(device="cuda").manual_seed(7)
    res = []
    for fn, cast in ((sandwich_norm_fn, lambda v: v.detach().clone()), (sandwich_norm_ref, lambda v: v.detach().double())):
        leaf = {k: None if v is None else cast(v).requires_grad_() for k, v in t.items()}
        y, s = fn(**leaf, **kw)
        if not res:
            dy, ds = (torch.randn(y.shape, generator=r, device="cuda").to(o.dtype) for o in (y, s))
        names = [k for k in leaf if leaf[k] is not None]
        grads = torch.autograd.grad((y, s), [leaf[k] for k in names], (dy.to(y.dtype), ds.to(s.dtype)))
        res.append((y, s, dict(zip(names, grads))))
    (y, s, g), (y2, s2, g2) = res
    close(y, y2, TOL[y.dtype] * tol_scale, "y")
    close(s, s2, TOL[s.dtype] * tol_scale, "residual_out")
    for k in g:
        assert g[k].dtype == t[k].dtype and g[k].shape == t[k].shape
        terms = 0.0
        if dx_cancels and k == "x":
            u = {n: v.double() for n, v in t.items()}
            s1 = u["gate"] * g2["residual"] / kw["residual_scale"] * u["post_weight"]
            terms = (s1 / u["x"].std(-1, correction=0, keepdim=True)).abs().max().item()
        off, top = (g[k].double() - g2[k]).abs().max().item(), max(g2[k].abs().max().item(), terms)
        assert off <= TOL[t[k].dtype] * tol_scale * top, f"d{k}: off by {off:.3e} of {top:.3e}"


@pytest.mark.parametrize("change, message", [
    (lambda t: {**t, "x": t["x"].double()}, "x must be"),
    (lambda t: {**t, "residual": t["residual"][:1]}, "residual"),
    (lambda t: {**t, "residual": t["residual"].half()}, "residual"),
    (lambda t: {**t, "post_weight": t["post_weight"][:3]}, "weights"),
    (lambda t: {**t, "pre_weight": None}, "required"),
    (lambda t: {**t, "gate": torch.ones(3, 1, 8)}, "gate must be"),
    (lambda t: {**t, "gate": torch.ones(1, 5, 8)}, "gate must be"),
    (lambda t: {**t, "gate": torch.ones(2, 8)}, "gate must"),
    (lambda t: t, "GPU"),
])
def test_refusals(change, message):
    with pytest.raises(RuntimeError, match=message):
        sandwich_norm_fn(**change(make((2, 5, 8), torch.float32, torch.float32, device="cpu")))


def test_rows_longer_than_8192_are_refused():
    t = make((1, 8193), torch.float32, torch.float32, device="cpu")
    with pytest.raises(RuntimeError, match="8192"):
        sandwich_norm_fn(**t)


def test_rows_beyond_32_bits_are_refused():
    t = make((1, 2), torch.float32, torch.float32, device="cpu")
    t["x"], t["residual"] = (t[k].expand(2**32 + 3, 2) for k in ("x", "residual"))
    with pytest.raises(RuntimeError, match="2\\^31"):
        sandwich_norm_fn(**t)


def test_c_entry_refuses():
    import ctypes

    import vms_hip
    L = vms_hip.lib()
    P = vms_hip.SandwichNormParams()
    assert L.vms_sandwich_norm_fwd(None, None) < 0 and L.vms_sandwich_norm_bwd(None, None) < 0
    assert L.vms_sandwich_norm_fwd(ctypes.byref(P), None) < 0 and b"empty" in L.vms_last_error()
    assert L.vms_sandwich_norm_bwd_workspace_bytes(ctypes.byref(P)) == 0
    P.rows, P.cols = 4, 9000
    assert L.vms_sandwich_norm_fwd(ctypes.byref(P), None) < 0 and b"8192" in L.vms_last_error()
    P.cols = 16
    assert L.vms_sandwich_norm_fwd(ctypes.byref(P), None) < 0 and b"required" in L.vms_last_error()
    P.x = P.post_weight = P.pre_weight = P.gate = 256
    P.rows_per_gate = 3
    assert L.vms_sandwich_norm_fwd(ctypes.byref(P), None) < 0 and b"rows_per_gate" in L.vms_last_error()
    P.rows_per_gate = 2
    P.stats = 260
    assert L.vms_sandwich_norm_fwd(ctypes.byref(P), None) < 0 and b"stats" in L.vms_last_error()


def test_c_workspace_size_of_bad_gate_rows():
    """0 for a block that the launch refuses, no division by zero (in a process of its own: that ended it)"""
    import subprocess
    import sys
    code = ("import ctypes, vms_hip\n"
            "L, P = vms_hip.lib(), vms_hip.SandwichNormParams()\n"
            "P.rows, P.cols, P.gate = 4, 16, 256\n"
            "got = []\n"
            "for n in (0, 1, 2, 3, 4, 8, 2**40):\n"
            "    P.rows_per_gate = n\n"
            "    got.append(L.vms_sandwich_norm_bwd_workspace_bytes(ctypes.byref(P)) > 0)\n"
            "print(got)")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, env={**os.environ, "PYTHONPATH": os.pathsep.join(sys.path)})
    assert r.returncode == 0 and r.stdout.strip() == "[False, True, True, False, True, False, False]", (r.returncode, r.stdout, r.stderr)


def test_an_empty_batch_with_a_gate_per_entry_is_no_division_by_zero():
    t = make((0, 5, 32), torch.float32, torch.float32, gate="batch", device="cpu")
    with pytest.raises(RuntimeError, match="GPU"):
        sandwich_norm_fn(**t)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(0, 5, 32), (3, 0, 32)])
@pytest.mark.parametrize("gate", ["none", "channel", "ones", "batch", "token"])
def test_empty_rows_with_every_gate(gate, shape):
    t = {k: v.requires_grad_() for k, v in make(shape, torch.bfloat16, torch.float32, gate=gate).items()}
    y, s = sandwich_norm_fn(**t)
    assert y.shape == s.shape == shape and s.dtype == torch.float32
    for k, g in zip(t, torch.autograd.grad(y.float().sum() + s.sum(), list(t.values()))):
        assert g.shape == t[k].shape and (g == 0).all(), k


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("n", [2, 7, 8, 100, 500, 512, 513, 768, 1024, 1025, 2048, 2052, 4096, 4100, 8192])
def test_columns(n, rms, dtype):
    compare(make((2, 11, n), dtype, dtype, gate="channel", seed=n), dx_cancels=n == 2 and not rms, is_rms_norm=rms, residual_scale=0.7)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("res32", [False, True])
@pytest.mark.parametrize("gate, gate_dtype", [("none", None), ("channel", torch.float32), ("ones", torch.bfloat16), ("batch", torch.bfloat16),
                                              ("batch", torch.float32), ("token", torch.float16), ("token", torch.float32)])
def test_gates_and_streams(gate, gate_dtype, res32, dtype):
    for bias in (False, True):
        compare(make((3, 37, 264), dtype, torch.float32 if res32 else dtype, bias=bias, gate=gate, gate_dtype=gate_dtype), is_rms_norm=not bias)


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [64, 1100, 4100])
@pytest.mark.parametrize("b, l", [(1, 1), (700, 3), (513, 1), (1200, 2), (2, 1500), (1, 5000)])
def test_group_sizes(b, l, cols):
    """few long gate groups (shared by workgroups), many short ones (walked whole), one row"""
    if b * l * cols > 6e6:
        l = max(1, l // 4)
    compare(make((b, l, cols), torch.bfloat16, torch.float32, gate="batch", gate_dtype=torch.bfloat16), is_rms_norm=True)


@pytest.mark.gpu
@pytest.mark.parametrize("b, l, cols", [(1100, 90, 16), (2100, 90, 8), (300, 50, 700), (4800, 2, 3), (70, 4, 3000)])
def test_group_counts_on_both_sides_of_the_plan(b, l, cols):
    """more groups than workgroups, shared and walked whole; few wide short ones"""
    compare(make((b, l, cols), torch.bfloat16, torch.float32, gate="batch", gate_dtype=torch.bfloat16))


@pytest.mark.gpu
@pytest.mark.parametrize("weight_dtype", [torch.float16, torch.bfloat16])
def test_weight_types_and_no_residual(weight_dtype):
    compare(make((2, 30, 96), torch.bfloat16, None, gate="channel", weight_dtype=weight_dtype))
    compare(make((60, 96), torch.float16, None, gate="none", weight_dtype=weight_dtype))
    x = make((2, 3, 16), torch.bfloat16, None)
    assert sandwich_norm_fn(**x, residual_in_fp32=True)[1].dtype == torch.float32 and sandwich_norm_fn(**x)[1].dtype == torch.bfloat16


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(dtype):
    t = make((2, 50, 72), dtype, dtype, gate="batch", gate_dtype=dtype)
    want = sandwich_norm_fn(**t)
    wide = torch.zeros(2, 50, 161, dtype=dtype, device="cuda")
    wide[..., 1:73], wide[..., 80:152] = t["x"], t["residual"]
    cut = {**t, "x": wide[..., 1:73], "residual": wide[..., 80:152], "gate": torch.cat([t["gate"]] * 2, -1)[..., :72]}
    turned = {**t, "x": t["x"].transpose(0, 1).contiguous().transpose(0, 1), "residual": t["residual"].mT.contiguous().mT}
    for other in (cut, turned):
        assert all(torch.equal(a, b) for a, b in zip(want, sandwich_norm_fn(**other)))
    leaf = {k: v.clone().requires_grad_() for k, v in t.items()}
    sandwich_norm_fn(**leaf)[0].sum().backward()      # an expanded gradient, and none for residual_out
    leaf2 = {k: v.double().requires_grad_() for k, v in t.items()}
    sandwich_norm_ref(**leaf2)[0].sum().backward()
    # the sum over a normed row weighted by nothing but pre_weight nearly cancels in dx: held to the size of what it is the difference of
    close(leaf["pre_weight"].grad, leaf2["pre_weight"].grad, 2e-5)
    close(leaf["pre_bias"].grad, leaf2["pre_bias"].grad, 2e-5)


@pytest.mark.gpu
def test_gradient_of_one_output_alone():
    t = make((2, 9, 40), torch.float32, torch.float32, gate="token")
    for which in (0, 1):
        a = {k: v.clone().requires_grad_() for k, v in t.items()}
        b = {k: v.double().requires_grad_() for k, v in t.items()}
        ga = torch.autograd.grad(sandwich_norm_fn(**a)[which].square().sum(), list(a.values()), allow_unused=True)
        gb = torch.autograd.grad(sandwich_norm_ref(**b)[which].square().sum(), list(b.values()), allow_unused=True)
        for k, u, v in zip(a, ga, gb):
            if v is not None:
                close(u, v, 4e-5, k)


@pytest.mark.gpu
def test_differences():
    """directional differences in fp32: f is a sum of 40 * 48 terms of size 1 computed to ~1e-7 each, h = 1e-2: rounding 5e-6 / 2 h = 2.5e-4"""
    t = make((2, 20, 48), torch.float32, torch.float32, gate="batch")
    r = torch.Generator(device="cuda").manual_seed(3)
    dy, ds = (torch.randn(t["x"].shape, generator=r, device="cuda").double() for _ in range(2))

    def f(v):
        y, s = sandwich_norm_fn(**v, residual_scale=1.3)
        return (y.double() * dy).sum() + (s.double() * ds).sum()

    leaf = {k: v.clone().requires_grad_() for k, v in t.items()}
    grads = dict(zip(leaf, torch.autograd.grad(f(leaf), list(leaf.values()))))
    for n in t:
        d = torch.randn(t[n].shape, generator=r, device="cuda")
        diff = ((f({**t, n: t[n] + 1e-2 * d}) - f({**t, n: t[n] - 1e-2 * d})) / 2e-2).item()
        got = (grads[n].double() * d).sum().item()
        assert abs(diff - got) <= 1e-2 * grads[n].norm().item() + 1e-3, (n, diff, got)


@pytest.mark.gpu
def test_equals_the_unfused_norms():
    """with a gate of one it is rms_norm_fn, then rms_norm_fn with the residual (fp32: no rounding between them)"""
    t = make((3, 17, 256), torch.float32, torch.float32, bias=False)
    y, s = sandwich_norm_fn(**t, is_rms_norm=True)
    h = rms_norm_fn(t["x"], t["post_weight"], None, eps=1e-6)
    y2, s2 = rms_norm_fn(h, t["pre_weight"], None, residual=t["residual"], prenorm=True, eps=1e-6)
    close(y, y2, 4e-6)
    close(s, s2, 4e-6)
    t = make((3, 17, 256), torch.float32, torch.float32)
    y, s = sandwich_norm_fn(**t)
    h = layer_norm_fn(t["x"], t["post_weight"], t["post_bias"])
    y2, s2 = layer_norm_fn(h, t["pre_weight"], t["pre_bias"], residual=t["residual"], prenorm=True)
    close(y, y2, 8e-6)
    close(s, s2, 8e-6)


@pytest.mark.gpu
def test_zero_rows_and_constant_rows():
    """an all-zero block output (rstd = eps^-1/2), a constant one (layer norm leaves nothing), a gate that drops whole entries"""
    t = make((4, 6, 64), torch.float32, torch.float32, gate="batch")
    t["x"][0], t["x"][1], t["gate"][2] = 0, 3.0, 0
    compare(t, tol_scale=4)   # rstd = 1000 multiplies the rounding of a mean that should be exact: 1000 * 3 * 2^-24 = 1.8e-4 of post_bias' size is no part of y's scale here
    y, s = sandwich_norm_fn(**t)
    assert torch.equal(s[2], t["residual"][2])


@pytest.mark.gpu
def test_empty_rows():
    t = make((0, 5, 32), torch.bfloat16, torch.float32)
    y, s = sandwich_norm_fn(**t)
    assert y.shape == (0, 5, 32) and s.dtype == torch.float32


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    t = make((2, 40), torch.bfloat16, torch.bfloat16)
    want = sandwich_norm_fn(**t)
    far = dict(t)
    for k in ("x", "residual"):
        far[k] = torch.empty(2**31 + 8 + 40, dtype=torch.bfloat16, device="cuda").as_strided((2, 40), (2**31 + 8, 1))
        far[k].copy_(t[k])
    assert all(torch.equal(a, b) for a, b in zip(want, sandwich_norm_fn(**far)))


@pytest.mark.gpu
def test_captured_and_same_bits():
    t = make((4, 100, 768), torch.bfloat16, torch.float32, gate="batch", gate_dtype=torch.bfloat16)
    static = {k: v.clone().requires_grad_() for k, v in t.items()}
    dy = torch.randn_like(t["x"])

    def go(v):
        y, s = sandwich_norm_fn(**v)
        return [y, s, *torch.autograd.grad((y, s), list(v.values()), (dy, s.detach()))]

    want = go({k: v.clone().requires_grad_() for k, v in t.items()})
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert all(torch.equal(a, b) for a, b in zip(want, go(static)))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = go(static)
    for _ in range(3):
        graph.replay()
        again = go({k: v.clone().requires_grad_() for k, v in t.items()})
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.gpu
def test_a_block_of_them():
    """as they are used together: pre-normed tokens -> projections -> gated delta rule -> projection -> sandwich norm, forward and backward in fp32,
    against the same block on the plain forms in 64 bits"""
    from mamba_ssm.ops.gated_delta_rule import gated_delta_rule_ref
    b, l, n, h, d = 2, 70, 64, 2, 32
    r = torch.Generator(device="cuda").manual_seed(11)
    randn = lambda *s: torch.randn(*s, generator=r, device="cuda")  # noqa: E731
    w = {"in": 0.15 * randn(n, 3 * h * d), "gb": 0.1 * randn(n, 2 * h), "out": 0.15 * randn(h * d, n), "w1": 1 + 0.1 * randn(n), "w2": 1 + 0.1 * randn(n),
         "gate": 0.5 + 0.1 * randn(n), "x": randn(b, l, n), "res": randn(b, l, n)}
    lens = torch.tensor([70, 33], dtype=torch.int32, device="cuda")
    dy = randn(b, l, n)

    def block(w, delta, sandwich):
        q, k, v = (w["x"] @ w["in"]).view(b, l, 3, h, d).unbind(2)
        q, k = (t / (t.square().sum(-1, keepdim=True) + 1e-6).sqrt() for t in (q, k))
        g, beta = (w["x"] @ w["gb"]).view(b, l, 2, h).unbind(2)
        o = sum(delta(q, k, v, -torch.nn.functional.softplus(g), beta.sigmoid(), reverse=rev, seq_lens=lens) for rev in (False, True))
        return sandwich(o.reshape(b, l, h * d) @ w["out"], w["res"], w["w1"], w["w2"], gate=w["gate"], residual_scale=0.9, is_rms_norm=True)

    def grads(w, *fns):
        w = {k: v.clone().requires_grad_() for k, v in w.items()}
        y, s = block(w, *fns)
        mask = (torch.arange(l, device="cuda")[None] < lens[:, None])[..., None]
        return [y * mask, s, *torch.autograd.grad((y * mask * dy.to(y.dtype)).sum() + s.square().sum() * 0.1, list(w.values()))]

    got = grads(w, gated_delta_rule_fn, sandwich_norm_fn)
    want = grads({k: v.double() for k, v in w.items()}, gated_delta_rule_ref, sandwich_norm_ref)
    for name, a, b_ in zip(["y", "s", *w], got, want):
        # padded tokens have a zero block output: 1 / deviation = 1000 there, which multiplies what the fp32 products leave
        close(a, b_, 4e-4, name)


@pytest.mark.gpu
@pytest.mark.parametrize("gate", ["none", "channel", "ones", "batch", "token"])
def test_compiled_and_ctypes_calls_are_one(gate, monkeypatch):
    import vms_hip
    ext = vms_hip.ext()
    assert ext is not None
    t = make((3, 20, 136), torch.bfloat16, torch.float32, gate=gate, gate_dtype=torch.float16, weight_dtype=torch.bfloat16)
    runs = []
    for use in (ext, None):
        monkeypatch.setattr(vms_hip, "_ext", use)
        leaf = {k: v.clone().requires_grad_() for k, v in t.items()}
        y, s = sandwich_norm_fn(**leaf, residual_scale=0.6)
        runs.append([y, s, *torch.autograd.grad((y, s), list(leaf.values()), (t["x"], s.detach()))])
        runs[-1] += [*sandwich_norm_fn(**{**t, "residual": None}, is_rms_norm=True)]
        g, = torch.autograd.grad(sandwich_norm_fn(**leaf)[1].square().sum(), leaf["x"], create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.float().sum().backward()
    assert all(torch.equal(a, b) and a.dtype == b.dtype for a, b in zip(*runs))
