"""mamba_ssm.ops.gated_delta_rule -- the gated delta rule, a linear recurrence over tokens with a matrix state per head, beside
selective_scan_fn (whole sequences, forward and backward) and selective_state_update (one new token).

Per batch entry and head, S (dk, dv), a_t = exp(g_t):
    S' = a_t S_{t-1};  u_t = beta_t (v_t - S'^T k_t);  S_t = S' + k_t u_t^T;  out_t = scale S_t^T q_t

The functions run csrc/gated_delta_*.hip and have no CPU path; the *_ref functions are the recurrence in plain PyTorch and run anywhere."""
import torch

import vms_hip as _k


def _check(cond, msg):
    if not cond:
        raise RuntimeError("gated_delta_rule: " + msg)


def _unit_last(t):
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _check_inputs(q, k, v, g, beta, lead):
    """lead: the axes before the heads (batch[, seqlen])"""
    _check(q.shape == k.shape and q.dim() == lead + 2 and v.dim() == lead + 2, "q, k (..., heads_k, dk) and v (..., heads, dv) expected")
    _check(q.shape[:lead] == v.shape[:lead], "q, k and v must agree in batch and length")
    _check(k.shape[lead] > 0 and v.shape[lead] % k.shape[lead] == 0, "the heads of v must be a multiple of the heads of q and k")
    _check(g.shape == v.shape[:-1] and beta.shape == g.shape, "g and beta must have the shape of v without its last axis")
    _check(1 <= k.shape[-1] <= 128, "key heads of 1 to 128 are supported")
    _check(1 <= v.shape[-1] <= 4096, "value heads of 1 to 4096 are supported")
    _check(max(v.shape) < 2 ** 31, "axes of less than 2^31 are supported")
    _check(q.dtype == v.dtype and k.dtype == v.dtype, "q, k and v must have one dtype")
    _check(v.dtype in (torch.float32, torch.float16, torch.bfloat16), "fp32, fp16 or bf16 expected")
    _check(g.dtype == beta.dtype and g.dtype in (v.dtype, torch.float32), "g and beta must have one dtype: fp32 or that of v")
    for t in (q, k, g, beta):
        _check(t.device == v.device, "all tensors must be on one device")


def _check_gpu(v):
    _check(v.is_cuda, "tensors must be on a GPU (no CPU path in this library)")


def _compiled(name, on_gpu):
    """the compiled binding's form of a call (the same checks and launches), None where it is not built"""
    ext = _k.ext() if on_gpu else None
    return getattr(ext, name, None)


class GatedDeltaRuleFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, beta, initial_state, scale, reverse, seq_lens, return_final_state):
        for_backward = any(ctx.needs_input_grad)
        q, k, v = _unit_last(q), _unit_last(k), _unit_last(v)
        batch, seqlen, heads, dv = v.shape
        dk = k.shape[-1]
        out = torch.empty(v.shape, dtype=v.dtype, device=v.device)
        final = torch.empty((batch, heads, dk, dv), dtype=torch.float32, device=v.device) if return_final_state else None
        s0 = initial_state.contiguous() if initial_state is not None else None
        ws = _k.gated_delta_fwd(q, k, v, g, beta, scale, s0, seq_lens, reverse, out, final, for_backward)
        if for_backward:
            ctx.save_for_backward(q, k, v, g, beta, seq_lens, ws)
            ctx.meta = (scale, reverse, initial_state is not None, initial_state is not None or return_final_state)
            ctx.set_materialize_grads(False)
        return out, final

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dfinal):
        q, k, v, g, beta, seq_lens, ws = ctx.saved_tensors
        scale, reverse, has_state, states = ctx.meta
        dout = torch.zeros_like(v) if dout is None else _unit_last(dout.to(v.dtype))
        dfinal = dfinal.float().contiguous() if dfinal is not None else None
        new = lambda t: torch.empty(t.shape, dtype=t.dtype, device=t.device)  # noqa: E731
        dq, dk, dv, dg, dbeta = new(q), new(k), new(v), new(g), new(beta)
        ds = torch.empty((v.shape[0], v.shape[2], k.shape[-1], v.shape[-1]), dtype=torch.float32, device=v.device) if has_state else None
        _k.gated_delta_bwd(q, k, v, g, beta, scale, seq_lens, reverse, states, ws, dout, dfinal, dq, dk, dv, dg, dbeta, ds)
        return dq, dk, dv, dg, dbeta, ds, None, None, None, None


def gated_delta_rule_fn(q, k, v, g, beta, scale=None, initial_state=None, return_final_state=False, reverse=False, seq_lens=None):
    """q, k (batch, seqlen, heads_k, dk), v (batch, seqlen, heads, dv), one dtype (fp32, fp16, bf16), any strides (a copy only where the last
    axis is strided); head h of v reads head h // (heads // heads_k) of q and k.  g (log decay, <= 0), beta (batch, seqlen, heads): that
    dtype or fp32.  scale: default dk ** -0.5.  1 <= dk <= 128.
    initial_state (batch, heads, dk, dv) fp32.  reverse=True: right to left, as in selective_scan.  seq_lens (batch,) integers on the
    device: the valid tokens of each batch entry, first in memory in either direction (values are clamped to 0 .. seqlen); the rest is padding
    that leaves the state alone, gives 0 and receives gradient 0.  Tokens are worked on 64 at a time: a NaN or infinity in a valid one reaches
    the outputs of its whole group of 64 and of what follows, none of the groups before.  batch, heads <= 65535, seqlen <= 2^30,
    batch * heads * ceil(dv / 32) < 2^23 (half of it for training in fp32).
    States are as exact as fp32 sums are, whatever q, k and v are; so are all gradients with an initial or a final state, or with fp32 q, k, v.  Without
    either, fp16 and bf16 gradients are carried to 2^-16 on the way, and so are fp32 gates' beside them.
    -> out (batch, seqlen, heads, dv), with return_final_state (out, final_state fp32).  Differentiable once in q, k, v, g, beta, initial_state."""
    fast = _compiled("gated_delta_rule", v.is_cuda and v.numel())
    if fast is not None:
        r = fast(q, k, v, g, beta, scale, initial_state, return_final_state, reverse, seq_lens)
        return tuple(r) if return_final_state else r[0]
    _check_inputs(q, k, v, g, beta, 2)
    batch, seqlen, heads, dv = v.shape
    dk = k.shape[-1]
    if initial_state is not None:
        _check(tuple(initial_state.shape) == (batch, heads, dk, dv) and initial_state.dtype == torch.float32 and initial_state.device == v.device,
               "initial_state must be fp32 (batch, heads, dk, dv) on the device of v")
    if seq_lens is not None:
        _check(tuple(seq_lens.shape) == (batch,) and seq_lens.device == v.device and seq_lens.dtype in (torch.int32, torch.int64),
               "seq_lens must be int32 or int64 (batch,) on the device of v")
    _check_gpu(v)
    if seq_lens is not None:
        # clamped before the narrowing: a 64-bit length must not wrap
        seq_lens = seq_lens.clamp(0, seqlen).to(torch.int32).contiguous() if seq_lens.dtype == torch.int64 else seq_lens.contiguous()
    scale = dk ** -0.5 if scale is None else float(scale)
    if v.numel() == 0:   # nothing to walk over: the state passes through, the other gradients are 0
        zero = 0 * sum(t.float().sum() for t in (q, k, v, g, beta))   # (a number where the state is not empty: then these are)
        s = torch.zeros((batch, heads, dk, dv), dtype=torch.float32, device=v.device) if initial_state is None else initial_state
        out = v + (zero + 0 * s.sum()).to(v.dtype)
        return (out, s + zero) if return_final_state else out
    out, final = GatedDeltaRuleFn.apply(q, k, v, g, beta, initial_state, scale, reverse, seq_lens, return_final_state)
    return (out, final) if return_final_state else out


def gated_delta_rule_ref(q, k, v, g, beta, scale=None, initial_state=None, return_final_state=False, reverse=False, seq_lens=None):
    """The recurrence token by token in fp32 (fp64 for fp64 inputs); arguments and results of gated_delta_rule_fn."""
    batch, seqlen, heads, dv = v.shape
    dk, rep = k.shape[-1], v.shape[2] // k.shape[2]
    scale = dk ** -0.5 if scale is None else scale
    acc = torch.float64 if v.dtype == torch.float64 else torch.float32
    state_dtype = acc
    q, k = (t.to(acc).repeat_interleave(rep, 2) for t in (q, k))
    lens = [seqlen] * batch if seq_lens is None else [min(max(int(n), 0), seqlen) for n in seq_lens]
    outs, finals = [], []
    for b in range(batch):
        S = torch.zeros(heads, dk, dv, dtype=acc, device=v.device) if initial_state is None else initial_state[b].to(acc)
        rows = [torch.zeros(heads, dv, dtype=acc, device=v.device)] * seqlen
        for i in range(lens[b]):
            t = lens[b] - 1 - i if reverse else i
            S = S * g[b, t].to(acc).exp()[:, None, None]
            u = beta[b, t].to(acc)[:, None] * (v[b, t].to(acc) - (S * k[b, t][:, :, None]).sum(1))
            S = S + k[b, t][:, :, None] * u[:, None, :]
            rows[t] = scale * (S * q[b, t][:, :, None]).sum(1)
        outs.append(torch.stack(rows) if seqlen else v.new_zeros(0, heads, dv, dtype=acc))
        finals.append(S)
    out = torch.stack(outs).to(v.dtype)
    return (out, torch.stack(finals).to(state_dtype)) if return_final_state else out


def _separate_states(state):
    """(batch, heads) states that each stand for themselves: (dk, dv) contiguous, none on top of another"""
    batch, heads, dk, dv = state.shape
    if not (dv == 1 or state.stride(3) == 1) or not (dk == 1 or state.stride(2) == dv):
        return False
    least = dk * dv
    for stride, n in sorted((state.stride(i), state.shape[i]) for i in (0, 1) if state.shape[i] > 1):
        if stride < least:
            return False
        least = stride * n
    return True


def gated_delta_state_update(state, q, k, v, g, beta, scale=None):
    """One token.  state (batch, heads, dk, dv) [in/out], fp32, fp16 or bf16, each (dk, dv) contiguous; q, k (batch, heads_k, dk), v (batch, heads, dv),
    one dtype; g, beta (batch, heads), that dtype or fp32; scale: default dk ** -0.5 -> out (batch, heads, dv).  The arithmetic is fp32; a
    16-bit state is rounded as it is stored, out is computed before that rounding.  Not differentiable.  batch * heads * ceil(dv / 32) < 2^24."""
    fast = _compiled("gated_delta_state_update", v.is_cuda)
    if fast is not None:
        return fast(state, q, k, v, g, beta, scale)
    _check_inputs(q, k, v, g, beta, 1)
    _check(state.dim() == 4 and tuple(state.shape) == (*v.shape[:2], k.shape[-1], v.shape[-1]), "state must be (batch, heads, dk, dv)")
    _check(state.dtype in (torch.float32, torch.float16, torch.bfloat16) and state.device == v.device, "state must be fp32, fp16 or bf16 on the device of v")
    _check(_separate_states(state), "the (dk, dv) states must be contiguous and must not overlap: they are updated in place")
    _check(not (torch.is_grad_enabled() and any(t.requires_grad for t in (state, q, k, v, g, beta))),
           "the single-token step has no gradient: call it under torch.no_grad(), or gated_delta_rule_fn")
    _check_gpu(v)
    out = torch.empty(v.shape, dtype=v.dtype, device=v.device)
    if v.numel():
        _k.gated_delta_step(state, _unit_last(q), _unit_last(k), _unit_last(v), g, beta, k.shape[-1] ** -0.5 if scale is None else scale, out)
        torch.autograd.graph.increment_version(state)
    return out


def gated_delta_state_update_ref(state, q, k, v, g, beta, scale=None):
    """The same in plain PyTorch (fp32, or fp64 for fp64 inputs); runs anywhere."""
    acc = torch.float64 if v.dtype == torch.float64 else torch.float32
    rep = v.shape[1] // k.shape[1]
    q, k = (t.to(acc).repeat_interleave(rep, 1) for t in (q, k))
    S = state.to(acc) * g.to(acc).exp()[..., None, None]
    u = beta.to(acc)[..., None] * (v.to(acc) - (S * k[..., None]).sum(-2))
    S = S + k[..., None] * u[..., None, :]
    state.copy_(S)
    return ((k.shape[-1] ** -0.5 if scale is None else scale) * (S * q[..., None]).sum(-2)).to(v.dtype)
