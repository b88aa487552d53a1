"""Normalisations a neuron can apply between its synaptic input and its dynamics
(counterpart of neuron/norm.py in the reference: MeanOnlyBatchNorm :9-95, WgtScaleBatchNorm :98-230).

Plain torch modules, as in the reference: they run once per call on the [N, C, ..., T] tensor and are not part
of the time-sequential kernels.  A neuron that is given one of them hooks its weight quantiser into
``pre_hook_fx`` (neuron/base.py:127-141 in the reference).

``group_norm`` and ``GroupNorm`` are for tensors with the channels last (tokens, images) and run in slayer_group_norm_fwd / bwd
of libslayer_hip.so."""
import torch

from .. import _native as N


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
