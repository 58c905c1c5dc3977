"""mamba_ssm.ops.triton.layernorm over the gfx950 kernels (reference: Triton kernels,
mamba/mamba_ssm/ops/triton/layernorm.py:51-503; the module path is kept because task code imports it).

  y = norm(x + residual) * weight + bias ; with prenorm=True also the pre-norm sum, kept in fp32 when
  residual_in_fp32.  layer_norm_fn / rms_norm_fn / RMSNorm run csrc/layer_norm.hip through layer_norm_cuda
  (no CPU path, like the reference's Triton kernels); layer_norm_ref / rms_norm_ref are the reference's
  pure-PyTorch functions (:19-48) and run anywhere.
"""
import torch
import torch.nn.functional as F

import layer_norm_cuda
import vms_hip as _k


def layer_norm_ref(x, weight, bias, residual=None, eps=1e-6, prenorm=False, upcast=False):
    dtype = x.dtype
    if upcast:
        weight = weight.float()
        bias = bias.float() if bias is not None else None
        x = x.float()
        residual = residual.float() if residual is not None else residual
    if residual is not None:
        x = (x + residual).to(x.dtype)
    out = F.layer_norm(x.to(weight.dtype), x.shape[-1:], weight=weight, bias=bias, eps=eps).to(dtype)
    return out if not prenorm else (out, x)


def rms_norm_ref(x, weight, bias, residual=None, eps=1e-6, prenorm=False, upcast=False):
    dtype = x.dtype
    if upcast:
        weight = weight.float()
        bias = bias.float() if bias is not None else None
        x = x.float()
        residual = residual.float() if residual is not None else residual
    if residual is not None:
        x = (x + residual).to(x.dtype)
    rstd = torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + eps)
    out = x * rstd * weight
    if bias is not None:
        out = out + bias
    out = out.to(dtype)
    return out if not prenorm else (out, x)


def _rows(t):
    """(..., N) -> (M, N) with a unit column stride (a copy only when the last dim is strided)."""
    t2 = t.reshape(-1, t.shape[-1])
    return t2 if t2.stride(-1) == 1 else t2.contiguous()


class LayerNormFn(torch.autograd.Function):
    """Autograd node of the fused add + norm: same inputs, outputs and gradient slots as the reference's
    LayerNormFn (layernorm.py:380-461); the kernels live in csrc/layer_norm.hip."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual=None, eps=1e-6, prenorm=False, residual_in_fp32=False,
                is_rms_norm=False):
        shape = x.shape
        if residual is not None and residual.shape != shape:
            raise ValueError("residual must have the shape of x")
        x2 = _rows(x)
        res2 = _rows(residual) if residual is not None else None
        # the pre-norm sum is stored in the residual's dtype, or in fp32 on request when there is no residual
        sum_dtype = res2.dtype if res2 is not None else (torch.float32 if residual_in_fp32 else None)
        y2, mean, rstd, presum = layer_norm_cuda.fwd(x2, weight.contiguous(), bias.contiguous() if bias is not None else None,
                                                     eps, res2, residual_dtype=sum_dtype, is_rms_norm=is_rms_norm)
        if presum is None:  # nothing added, no dtype change: the sum is x itself
            presum = x2
        ctx.save_for_backward(presum, weight, bias, mean, rstd)
        ctx.meta = (shape, eps, is_rms_norm, residual is not None, prenorm, x2.dtype)
        y = y2.reshape(shape)
        return (y, presum.reshape(shape)) if prenorm else y

    @staticmethod
    def backward(ctx, dy, *more):
        presum, weight, bias, mean, rstd = ctx.saved_tensors
        shape, eps, is_rms, had_residual, prenorm, x_dtype = ctx.meta
        dy2 = _rows(dy)
        dsum = _rows(more[0]) if prenorm else None  # gradient that arrived through the prenorm output
        dx, dw, db, dres = layer_norm_cuda.bwd(dy2, presum, weight, bias, eps, mean, rstd, dsum, had_residual, is_rms,
                                               x_dtype=x_dtype)
        return (dx.reshape(shape), dw, db, dres.reshape(shape) if had_residual else None, None, None, None, None)


def layer_norm_fn(x, weight, bias, residual=None, eps=1e-6, prenorm=False, residual_in_fp32=False,
                  is_rms_norm=False):
    return LayerNormFn.apply(x, weight, bias, residual, eps, prenorm, residual_in_fp32, is_rms_norm)


def rms_norm_fn(x, weight, bias, residual=None, prenorm=False, residual_in_fp32=False, eps=1e-6,
                is_rms_norm=True):
    return LayerNormFn.apply(x, weight, bias, residual, eps, prenorm, residual_in_fp32, is_rms_norm)


class RMSNorm(torch.nn.Module):
    def __init__(self, hidden_size, eps=1e-5, device=None, dtype=None):
        factory_kwargs = {"device": device, "dtype": dtype}
        super().__init__()
        self.eps = eps
        self.weight = torch.nn.Parameter(torch.empty(hidden_size, **factory_kwargs))
        self.register_parameter("bias", None)
        self.reset_parameters()

    def reset_parameters(self):
        torch.nn.init.ones_(self.weight)

    def forward(self, x, residual=None, prenorm=False, residual_in_fp32=False):
        return rms_norm_fn(x, self.weight, self.bias, residual=residual, eps=self.eps, prenorm=prenorm,
                           residual_in_fp32=residual_in_fp32, is_rms_norm=True)


# ---- the norms around a residual block -----------------------------------------------------------------------
def sandwich_norm_ref(x, residual, post_weight, pre_weight, post_bias=None, pre_bias=None, gate=None, residual_scale=1.0,
                      residual_in_fp32=False, eps=1e-6, is_rms_norm=False):
    """sandwich_norm_fn in plain PyTorch (fp32, or fp64 for fp64 inputs); runs anywhere."""
    acc = torch.float64 if x.dtype == torch.float64 else torch.float32
    up = lambda t: t.to(acc) if t is not None else None  # noqa: E731

    def norm(z, weight, bias):
        if not is_rms_norm:
            z = z - z.mean(-1, keepdim=True)
        z = z * torch.rsqrt(z.square().mean(-1, keepdim=True) + eps) * up(weight)
        return z if bias is None else z + up(bias)

    r = norm(up(x), post_weight, post_bias)
    if gate is not None:
        r = r * up(gate)
    if residual is not None:
        r = r + residual_scale * up(residual)
    stream = residual.dtype if residual is not None else torch.float32 if residual_in_fp32 and acc == torch.float32 else x.dtype
    return norm(r, pre_weight, pre_bias).to(x.dtype), r.to(stream)


def _require(cond, msg):
    if not cond:
        raise RuntimeError("sandwich_norm_fn: " + msg)


class SandwichNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, post_weight, pre_weight, post_bias, pre_bias, gate, rows_per_gate, residual_scale, stream, eps, is_rms_norm):
        x2 = _rows(x)
        res2 = _rows(residual) if residual is not None else None
        gate2 = _rows(gate) if gate is not None else None
        fp32 = lambda t: t.float().contiguous() if t is not None else None  # noqa: E731
        par = (fp32(post_weight), fp32(post_bias), fp32(pre_weight), fp32(pre_bias))
        rows, cols = x2.shape
        y = torch.empty((rows, cols), dtype=x.dtype, device=x.device)
        out = torch.empty((rows, cols), dtype=stream, device=x.device)
        for_backward = any(ctx.needs_input_grad)
        stats = torch.empty((rows, 4), dtype=torch.float32, device=x.device) if for_backward else None
        _k.sandwich_norm_fwd(x2, res2, gate2, rows_per_gate, *par, y, out, stats, residual_scale, eps, is_rms_norm)
        if for_backward:
            ctx.save_for_backward(x2, res2, gate2, *par, stats)
            ctx.meta = (x.shape, None if gate is None else gate.shape, rows_per_gate, residual_scale, stream, eps, is_rms_norm,
                        [None if t is None else t.dtype for t in (post_weight, pre_weight, post_bias, pre_bias)])
            ctx.set_materialize_grads(False)
        return y.view(x.shape), out.view(x.shape)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dout):
        x, res, gate, *par, stats = ctx.saved_tensors
        shape, gate_shape, rows_per_gate, residual_scale, stream, eps, is_rms_norm, dtypes = ctx.meta
        dy = _rows(dy.to(x.dtype)) if dy is not None else None
        dout = _rows(dout.to(stream)) if dout is not None else None
        new = lambda t: torch.empty(t.shape, dtype=t.dtype, device=t.device) if t is not None else None  # noqa: E731
        dx, dres, dgate, dpost_w, dpost_b, dpre_w, dpre_b = new(x), new(res), new(gate), *(new(t) for t in par)
        _k.sandwich_norm_bwd(x, res, gate, rows_per_gate, *par, stats, stream, residual_scale, eps, is_rms_norm,
                             dy, dout, dx, dres, dgate, dpost_w, dpost_b, dpre_w, dpre_b)
        cast = lambda t, d: t.to(d) if t is not None else None  # noqa: E731
        return (dx.view(shape), dres.view(shape) if dres is not None else None, cast(dpost_w, dtypes[0]), cast(dpre_w, dtypes[1]),
                cast(dpost_b, dtypes[2]), cast(dpre_b, dtypes[3]), dgate.view(gate_shape) if dgate is not None else None,
                None, None, None, None, None)


def sandwich_norm_fn(x, residual, post_weight, pre_weight, post_bias=None, pre_bias=None, gate=None, residual_scale=1.0,
                     residual_in_fp32=False, eps=1e-6, is_rms_norm=False):
    """The norm after a block, its gate, the scaled residual add and the norm before the next block in one pass (csrc/sandwich_norm.hip;
    layer_norm_fn fuses the last two only):
        h = norm(x; post_weight, post_bias);  residual_out = residual_scale * residual + gate * h;  y = norm(residual_out; pre_weight, pre_bias)
    x (..., N) fp32, fp16 or bf16, N <= 8192; residual: the shape of x, its dtype or fp32, or None (zeros; the stream is then fp32 with
    residual_in_fp32, else x's dtype).  Weights and biases (N), any of the three dtypes.  gate, any of them too: (N) or (1, ..., 1, N) for all rows, (batch, 1,
    ..., 1, N) for each entry of x's first axis (its zero rows drop a residual branch), or the shape of x.  y is the norm of the sum before
    it is rounded to the stream's dtype.  -> (y, residual_out).  Differentiable once in every tensor."""
    N = x.shape[-1] if x.dim() else 0
    floats = (torch.float32, torch.float16, torch.bfloat16)
    _require(x.dim() >= 2 and x.dtype in floats, "x must be (..., N) in fp32, fp16 or bf16")
    _require(1 <= N <= 8192, "rows of 1 to 8192 are supported")
    if residual is not None:
        _require(residual.shape == x.shape and residual.dtype in (x.dtype, torch.float32), "residual must have the shape of x, and its dtype or fp32")
    for t in (post_weight, pre_weight, post_bias, pre_bias):
        _require(t is None or (tuple(t.shape) == (N,) and t.dtype in floats), "weights and biases must be (N,) in fp32, fp16 or bf16")
    _require(post_weight is not None and pre_weight is not None, "post_weight and pre_weight are required")
    rows = x.numel() // N
    _require(rows < 2 ** 31, "less than 2^31 rows are supported")
    rows_per_gate = 0
    if gate is not None:
        lead = tuple(gate.shape[:-1])
        _require(gate.dim() in (1, x.dim()) and gate.shape[-1] == N and gate.dtype in floats, "gate must be (N,) or have as many axes as x, in fp32, fp16 or bf16")
        if gate.shape == x.shape:
            rows_per_gate = 1
        elif all(n == 1 for n in lead):
            rows_per_gate = rows
        else:
            _require(lead[0] == x.shape[0] and all(n == 1 for n in lead[1:]), "gate must be (N,), (batch, 1, ..., 1, N) or of the shape of x")
            rows_per_gate = rows // max(x.shape[0], 1)   # (an empty batch has none)
    tensors = [t for t in (residual, post_weight, pre_weight, post_bias, pre_bias, gate) if t is not None]
    _require(all(t.device == x.device for t in tensors), "all tensors must be on one device")
    _require(x.is_cuda, "tensors must be on a GPU (no CPU path in this library)")
    if rows == 0:
        return sandwich_norm_ref(x, residual, post_weight, pre_weight, post_bias, pre_bias, gate, residual_scale, residual_in_fp32, eps, is_rms_norm)
    stream = residual.dtype if residual is not None else torch.float32 if residual_in_fp32 else x.dtype
    fast = getattr(_k.ext(), "sandwich_norm", None)   # the compiled binding's node: the same launches
    if fast is not None:
        return tuple(fast(x, residual, post_weight, pre_weight, post_bias, pre_bias, gate, rows_per_gate, residual_scale,
                          stream == torch.float32, eps, is_rms_norm))
    return SandwichNormFn.apply(x, residual, post_weight, pre_weight, post_bias, pre_bias, gate, rows_per_gate, float(residual_scale), stream,
                                float(eps), bool(is_rms_norm))
