"""Normalisations a neuron can apply between its synaptic input and its dynamics
(counterpart of neuron/norm.py in the reference: MeanOnlyBatchNorm :9-95, WgtScaleBatchNorm :98-230).

Plain torch modules, as in the reference: they run once per call on the [N, C, ..., T] tensor and are not part
of the time-sequential kernels.  A neuron that is given one of them hooks its weight quantiser into
``pre_hook_fx`` (neuron/base.py:127-141 in the reference).

``group_norm`` and ``GroupNorm`` are for tensors with the channels last (tokens, images) and run in slayer_group_norm_fwd / bwd
of libslayer_hip.so; ``residual_norm`` and ``ResidualNorm``, the norms behind a block and in front of the next one, in
slayer_residual_norm_fwd / bwd."""
import torch

from .. import _native as N
from ..utils.types import KeepsTypes


def _identity(x, descale=False):
    return x


class _FeatureNorm(torch.nn.Module):
    """Per-feature (axis 1) running mean with momentum; the first input fixes the feature count."""

    def __init__(self, num_features, momentum, pre_hook_fx):
        super().__init__()
        self.num_features = num_features
        self.momentum = momentum
        self.pre_hook_fx = _identity if pre_hook_fx is None else pre_hook_fx
        self.register_buffer('running_mean', torch.zeros(1 if num_features is None else num_features))
        self.update = True

    @property
    def bias(self):
        """The mean as the (negative) bias a hardware neuron would carry."""
        return -self.pre_hook_fx(self.running_mean, descale=True)

    def _mean(self, inp):
        """Batch mean per feature while training (and updating), else the running estimate; also says
        whether the batch statistics were used."""
        if self.num_features is None:
            self.num_features = inp.shape[1]
        if self.training and self.update is True:
            mean = torch.mean(inp.reshape(inp.shape[0], self.num_features, -1), dim=[0, 2])
            with torch.no_grad():
                self.running_mean = (1 - self.momentum) * self.running_mean + self.momentum * mean
            return mean, True
        return self.running_mean, False

    @staticmethod
    def _per_feature(v, inp):
        if not 2 <= inp.dim() <= 5:
            raise AssertionError(f'Found unexpected number of dims {inp.dim()} in input.')
        return v.reshape((1, -1) + (1,) * (inp.dim() - 2))


class MeanOnlyBatchNorm(_FeatureNorm):
    """Subtracts the per-feature mean (batch mean while training, running mean otherwise); the
    subtracted value goes through ``pre_hook_fx`` first, so it can be quantised like a weight."""

    def __init__(self, num_features=None, momentum=0.1, pre_hook_fx=None):
        super().__init__(num_features, momentum, pre_hook_fx)

    def reset_parameters(self):
        self.running_mean.zero_()

    def forward(self, inp):
        mean, _ = self._mean(inp)
        return inp - self.pre_hook_fx(self._per_feature(mean, inp))


class WgtScaleBatchNorm(_FeatureNorm):
    """Mean subtraction plus a division by the standard deviation of the whole tensor rounded up to a power
    of two (exponent limited to +-``weight_exp_bits``), so that hardware can apply it as a shift."""

    def __init__(self, num_features=None, momentum=0.1, weight_exp_bits=3, eps=1e-5, pre_hook_fx=None):
        super().__init__(num_features, momentum, pre_hook_fx)
        self.weight_exp_bits = weight_exp_bits
        self.eps = eps
        self.register_buffer('running_var', torch.zeros(1))

    def reset_parameters(self):
        self.running_mean.zero_()
        self.running_var.zero_()

    def std(self, var):
        exponent = torch.ceil(torch.log2(torch.sqrt(var + self.eps)))
        return torch.pow(2., exponent.clamp(-self.weight_exp_bits, self.weight_exp_bits))

    @property
    def weight_exp(self):
        """Exponent of the equivalent weight scaling."""
        return torch.ceil(torch.log2(torch.sqrt(self.running_var + self.eps)))

    def forward(self, inp):
        mean, batch = self._mean(inp)
        if batch:
            var = torch.var(inp, unbiased=False)
            n = inp.numel() / inp.shape[1]
            with torch.no_grad():
                self.running_var = (1 - self.momentum) * self.running_var + self.momentum * var * n / (n + 1)
        else:
            var = self.running_var
        return (inp - self.pre_hook_fx(self._per_feature(mean, inp))) / self._per_feature(self.std(var), inp)


ACTIVATIONS = {None: 0, 'none': 0, 'relu': 1, 'silu': 2, 'gelu': 3}


def group_norm(input, num_groups, weight=None, bias=None, eps=1e-5, activation=None):
    """Group norm over the last axis with an activation behind it, in one operator: for each sample (first axis) the
    channels (last axis) are cut into ``num_groups`` groups of neighbours; a group is normalised over its channels and
    all positions between first and last axis, scaled, shifted and activated.

    Parameters
    ----------
    input : torch.Tensor
        float32 or bfloat16 GPU tensor [N, ..., C].
    num_groups : int
        divides C; N * num_groups at most 2**23 where a group reaches over more than one position.
    weight, bias : torch.Tensor or None
        C floating-point values each; None: 1 and 0.
    eps : float
    activation : None, 'none', 'relu', 'silu' or 'gelu' (with the error function)

    Returns
    -------
    torch.Tensor, contiguous, of the shape and type of ``input``.  Statistics, weights and their gradients are float32.
    """
    if activation not in ACTIVATIONS:
        raise ValueError(f'unknown activation {activation!r}: one of {list(ACTIVATIONS)}')
    N.require_elements(input)
    if input.dim() < 2:
        raise RuntimeError(f'expected a tensor [N, ..., C], got {input.dim()} axes')
    channels = input.shape[-1]
    if num_groups < 1 or channels < 1 or channels % num_groups:
        raise RuntimeError(f'{channels} channels cannot be cut into {num_groups} groups')
    if not eps >= 0:
        raise ValueError(f'eps has to be at least 0, got {eps}')
    for name, t in (('weight', weight), ('bias', bias)):
        if t is not None:
            if not torch.is_tensor(t) or t.shape != (channels,) or not t.is_floating_point():
                raise RuntimeError(f'{name}: expected {channels} floating-point values')
            if t.device != input.device:
                raise RuntimeError(f'tensors on different devices: {input.device} and {t.device}')
    weight = weight if weight is None else weight.float().contiguous()
    bias = bias if bias is None else bias.float().contiguous()
    code = ACTIVATIONS[activation]
    if N.wants_grad(*(t for t in (input, weight, bias) if t is not None)):
        return _GroupNorm.apply(input, weight, bias, num_groups, eps, code)
    return _norm_fwd(input.contiguous(), weight, bias, num_groups, eps, code, False)[0]


def _norm_sizes(input, groups):
    n, c = input.shape[0], input.shape[-1]
    return n, (input.numel() // (n * c) if n else 0), c, groups


def _norm_fwd(input, weight, bias, groups, eps, activation, keep):
    """(out, statistics or None): the means and then the scales of all groups."""
    dtype = N.ELEMENT_TYPES[input.dtype]
    sizes = _norm_sizes(input, groups)
    lib = N.lib()
    floats = lib.slayer_group_norm_workspace(dtype, *sizes, 0)
    if floats < 0:
        N.check(int(floats))
    out = torch.empty_like(input)
    stats = mean = scale = None
    if keep or floats:
        count = sizes[0] * groups
        stats = torch.empty(2 * count, dtype=torch.float32, device=input.device)
        mean = stats.data_ptr()
        scale = mean + 4 * count
    workspace = torch.empty(floats, dtype=torch.float32, device=input.device) if floats else None
    with N.device_guard(input.device):
        N.check(lib.slayer_group_norm_fwd(out.data_ptr(), mean, scale, input.data_ptr(), N.ptr(weight), N.ptr(bias), dtype, *sizes,
                                          eps, activation, N.ptr(workspace), floats, N.stream_handle()))
    return out, stats


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, input, weight, bias, groups, eps, activation):
        input = input.contiguous()
        out, stats = _norm_fwd(input, weight, bias, groups, eps, activation, True)
        ctx.save_for_backward(input, weight, bias, stats)
        ctx.args = (groups, activation)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_output):
        input, weight, bias, stats = ctx.saved_tensors
        groups, activation = ctx.args
        grad_output = grad_output.contiguous()
        dtype, sizes = N.ELEMENT_TYPES[input.dtype], _norm_sizes(input, groups)
        grad = torch.empty_like(input)
        need_weight, need_bias = weight is not None and ctx.needs_input_grad[1], bias is not None and ctx.needs_input_grad[2]
        channels, mean = sizes[2], stats.data_ptr()
        lib = N.lib()
        floats = lib.slayer_group_norm_workspace(dtype, *sizes, 1)
        if floats < 0:
            N.check(int(floats))
        sums = torch.empty((2, channels), dtype=torch.float32, device=input.device)
        workspace = torch.empty(floats, dtype=torch.float32, device=input.device)
        at = sums.data_ptr()
        with N.device_guard(input.device):
            N.check(lib.slayer_group_norm_bwd(grad.data_ptr(), at if need_weight else None, at + 4 * channels if need_bias else None,
                                              grad_output.data_ptr(), input.data_ptr(), mean, mean + 4 * sizes[0] * groups,
                                              N.ptr(weight), N.ptr(bias), dtype, *sizes, activation, workspace.data_ptr(), floats,
                                              N.stream_handle()))
        return grad, sums[0] if need_weight else None, sums[1] if need_bias else None, None, None, None


class GroupNorm(torch.nn.Module):
    """:func:`group_norm` with a trained weight and bias for each channel (``affine=False``: without)."""

    def __init__(self, num_groups, num_channels, eps=1e-5, affine=True, activation=None):
        super().__init__()
        if num_groups < 1 or num_channels < 1 or num_channels % num_groups:
            raise ValueError(f'{num_channels} channels cannot be cut into {num_groups} groups')
        if activation not in ACTIVATIONS:
            raise ValueError(f'unknown activation {activation!r}: one of {list(ACTIVATIONS)}')
        self.num_groups, self.num_channels, self.eps, self.activation = num_groups, num_channels, eps, activation
        self.weight = torch.nn.Parameter(torch.ones(num_channels)) if affine else None
        self.bias = torch.nn.Parameter(torch.zeros(num_channels)) if affine else None

    def forward(self, input):
        return group_norm(input, self.num_groups, self.weight, self.bias, self.eps, self.activation)

    def extra_repr(self):
        return f'{self.num_groups}, {self.num_channels}, eps={self.eps}, activation={self.activation}'


GATES = {None: 1, 'none': 1, 'sigmoid': 2, 'silu': 3}


def residual_norm(input, residual, weight=None, inner=None, gate=None, scale=None, activation='sigmoid', eps=1e-5, return_sum=True):
    """What stands between two blocks, in one operator: the norm of a block's result, its gate and scale, the residual stream, and the
    norm in front of the next block,

        total = residual + scale * act(gate) * inner * input / rms(input),    out = weight * total / rms(total),

    with rms(x) = sqrt(mean(x ** 2) + eps) over the last axis.

    Parameters
    ----------
    input : torch.Tensor
        float32 or bfloat16 GPU tensor [..., C], C at most 8192.  Rows that lie a fixed distance from each other (a part of a
        projection) are read where they lie, others are copied first; so for residual and gate.
    residual : torch.Tensor or None
        of the same shape and type, or float32 (a stream that is kept in float32 between bfloat16 blocks); None: 0.
    weight : torch.Tensor or None
        C floating-point values of the norm in front of the next block; None: there is none, and no ``out``.
    inner : torch.Tensor or None
        C floating-point values of the norm behind the block; None: there is none.
    gate : torch.Tensor or None
        of the shape and type of input.
    scale : torch.Tensor, float or None
        C floating-point values, or one number.
    activation : 'sigmoid', 'silu', None or 'none'
        of the gate.
    eps : float
    return_sum : bool
        whether ``total`` is wanted (always without a ``weight``).

    Returns
    -------
    (out, total), contiguous, of the types of input and residual (of input without one); ``out`` alone without ``return_sum``, ``total``
    alone without a ``weight``.  ``out`` is that of the sum before it is rounded to the type of ``total``.  Statistics, weights and their
    gradients are float32.
    """
    if activation not in GATES:
        raise ValueError(f'unknown activation {activation!r}: one of {list(GATES)}')
    if not eps >= 0:
        raise ValueError(f'eps has to be at least 0, got {eps}')
    device, _ = N.require_elements(input) if gate is None else N.require_elements(input, gate)
    shape = input.shape
    if len(shape) < 1 or not 1 <= shape[-1] <= 8192:
        raise RuntimeError(f'expected a tensor [..., C] with C up to 8192, got {tuple(shape)}')
    if gate is not None and gate.shape != shape:
        raise RuntimeError(f'gate: expected the shape {tuple(shape)}, got {tuple(gate.shape)}')
    if residual is not None:
        if not torch.is_tensor(residual) or residual.shape != shape or residual.dtype not in (input.dtype, torch.float32):
            raise RuntimeError(f'residual: expected a tensor {list(shape)} of {input.dtype} or torch.float32')
        if residual.device != device:
            raise RuntimeError(f'tensors on different devices: {device} and {residual.device}')
    factor = 1.0
    if scale is not None and not torch.is_tensor(scale):
        factor, scale = float(scale), None
    weight, inner, scale = (_parameter(name, t, shape[-1], device) for name, t in (('weight', weight), ('inner', inner), ('scale', scale)))
    tensors = (input, residual, gate, weight, inner, scale)
    args = (0 if gate is None else GATES[activation], float(eps), factor, return_sum or weight is None)
    if N.wants_grad(*tensors):
        out, total = _ResidualNorm.apply(*tensors, *args)
    else:
        out, total = _residual_fwd(*tensors, *args, False)[:2]
    if weight is None:
        return total
    return (out, total) if return_sum else out


def _parameter(name, t, channels, device):
    """``t`` as float32 and contiguous, or None."""
    if t is None:
        return None
    if not torch.is_tensor(t) or t.shape != (channels,) or not t.is_floating_point():
        raise RuntimeError(f'{name}: expected {channels} floating-point values')
    if t.device != device:
        raise RuntimeError(f'tensors on different devices: {device} and {t.device}')
    return t if t.dtype is torch.float32 and t.is_contiguous() else t.float().contiguous()


def _rows(x):
    """``x`` as rows of neighbouring elements (a view where it can be one), and how far they are apart."""
    if x is None:
        return None, 0
    channels = x.shape[-1]
    if not x.is_contiguous():
        x = x.reshape(x.numel() // channels, channels)
        if channels == 1 or x.stride(1) == 1:
            return x, x.stride(0)
        x = x.contiguous()
    return x, channels


def _residual_call(shape, input, residual, gate, weight, inner, scale, activation, eps, factor):
    """The structure of the C calls, and the tensors it describes."""
    kind, channels = N.ELEMENT_TYPES, shape[-1]
    (input, a), (residual, b), (gate, c) = _rows(input), _rows(residual), _rows(gate)
    dtype = kind[input.dtype]
    call = N.ResidualNorm(input.numel() // channels, channels, N.ptr(inner), N.ptr(weight), N.ptr(scale), dtype,
                          dtype if residual is None else kind[residual.dtype], activation, eps, factor, a, b, c)
    return call, input, residual, gate


def _residual_fwd(input, residual, gate, weight, inner, scale, activation, eps, factor, want_total, keep):
    device = input.device
    out = None if weight is None else N.empty_as(input)
    total = N.empty_as(input if residual is None else residual) if want_total else None
    call, input, residual, gate = _residual_call(input.shape, input, residual, gate, weight, inner, scale, activation, eps, factor)
    stats = torch.empty((call.rows, 2), dtype=torch.float32, device=device) if keep else None
    with N.device_guard(device):
        N.check(N.lib().slayer_residual_norm_fwd(N.ptr(out), N.ptr(total), N.ptr(stats), input.data_ptr(), N.ptr(residual), N.ptr(gate),
                                                 call, N.stream_handle()))
    return out, total, input, residual, gate, stats


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, input, residual, gate, weight, inner, scale, activation, eps, factor, want_total):
        ctx.shape, ctx.args = input.shape, (activation, eps, factor)
        out, total, *saved = _residual_fwd(input, residual, gate, weight, inner, scale, activation, eps, factor, want_total, True)
        ctx.save_for_backward(*saved, weight, inner, scale)
        ctx.set_materialize_grads(False)
        return out, total

    @staticmethod
    @N.once_differentiable
    def backward(ctx, grad_out, grad_total):
        if grad_out is None and grad_total is None:
            return (None,) * 10
        input, residual, gate, stats, weight, inner, scale = ctx.saved_tensors
        device, shape, need = input.device, ctx.shape, ctx.needs_input_grad
        call = _residual_call(shape, input, residual, gate, weight, inner, scale, *ctx.args)[0]
        grad_out, call.grad_out_stride = _rows(grad_out)
        grad_total, call.grad_total_stride = _rows(grad_total)
        grads = [torch.empty(shape, dtype=t.dtype, device=device) if wanted else None
                 for t, wanted in zip((input, residual, gate), need)]
        sums = [torch.empty_like(t) if wanted else None for t, wanted in zip((weight, inner, scale), need[3:])]
        lib, workspace, floats = N.lib(), None, 0
        if any(need[3:6]):
            floats = lib.slayer_residual_norm_workspace(call)
            if floats < 0:
                N.check(int(floats))
            workspace = torch.empty(floats, dtype=torch.float32, device=device)
        with N.device_guard(device):
            N.check(lib.slayer_residual_norm_bwd(*(N.ptr(g) for g in grads), N.ptr(sums[1]), N.ptr(sums[0]), N.ptr(sums[2]),
                                                 N.ptr(grad_out), N.ptr(grad_total), stats.data_ptr(), input.data_ptr(), N.ptr(residual),
                                                 N.ptr(gate), call, N.ptr(workspace), floats, N.stream_handle()))
        return (*grads, *sums, None, None, None, None)


class ResidualNorm(KeepsTypes):
    """:func:`residual_norm` with trained weights: ``inner`` and ``outer`` say which of the two norms there are, ``scale`` is the residual
    scale that every channel starts with (None: there is none), ``activation`` that of the gate, where ``forward`` is given one.  The
    weights are float32 whatever the type of the module (``.to(torch.bfloat16)``)."""

    def __init__(self, num_channels, inner=True, outer=True, scale=None, activation='sigmoid', eps=1e-5):
        super().__init__()
        if activation not in GATES:
            raise ValueError(f'unknown activation {activation!r}: one of {list(GATES)}')
        self.num_channels, self.activation, self.eps = num_channels, activation, eps
        self.weight = torch.nn.Parameter(torch.ones(num_channels)) if outer else None
        self.inner = torch.nn.Parameter(torch.ones(num_channels)) if inner else None
        self.scale = None if scale is None else torch.nn.Parameter(torch.full((num_channels,), float(scale)))

    def forward(self, input, residual=None, gate=None, return_sum=True):
        return residual_norm(input, residual, self.weight, self.inner, gate, self.scale, self.activation, self.eps, return_sum)

    def extra_repr(self):
        return (f'{self.num_channels}, inner={self.inner is not None}, outer={self.weight is not None}, '
                f'scale={self.scale is not None}, activation={self.activation}, eps={self.eps}')
