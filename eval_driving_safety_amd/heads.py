"""Fully connected layers on libadvengine's kernels: trained with a counter-based dropout, or served / attacked with four-bit weights.

``LinearDropout`` stands for Linear - Dropout (- ReLU) of a head in training (dynamic_vehicles/Model.py:24-27, driving_constraint/Model.py:21-23):
the product is torch's, bias + dropout + ReLU are one kernel (``ops.Dropout``), and the mask of step s under a seed is the same in every process.
``Mx4LinearLayer`` stands for a frozen Linear (- ReLU) whose weight is held in MXFP4 (``ops.Mx4Linear``): gradients flow to its input only, as
through every adopted layer."""
import threading
import types

import torch
import torch.nn as nn
import torch.nn.functional as F

_FIRST_USE = threading.Lock()


def layer_seed(seed, index):
    """another key for every dropout layer of a model"""
    return (int(seed) + index * 0x9E3779B97F4A7C15) % (1 << 64)


class _Counted:
    """dropout under ``seed`` whose every forward takes the next ``step``"""

    def _drop(self, y, bias=None, relu=False):
        from . import ops
        step = self.step
        if not isinstance(step, torch.Tensor):
            if y.is_cuda and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("%s: a captured step needs `step` as an int64 CUDA tensor (a number would give every replay the same mask)" % type(self).__name__)
            if torch._C._current_graph_task_id() != -1:            # inside a backward pass
                raise RuntimeError("%s: a forward recomputed in the backward pass needs `step` as an int64 tensor (the number has moved on: another mask)" % type(self).__name__)
            self.step = step + 1
        return ops.Dropout.apply(y, self.p, self.seed, step, bias, relu)


class LinearDropout(_Counted, nn.Linear):
    """``relu?(dropout(linear(x)))`` with ``nn.Linear``'s parameters and state-dict keys.  In training every forward takes the next ``step`` (a plain
    number: set it to go on where another run stopped); in eval there is no dropout.  Training needs a ROCm device.  For a step captured in a
    hipGraph set ``step`` to an int64 CUDA tensor of one element and move it on between the replays (a number would repeat one mask: refused).  The same
    where activations are recomputed in the backward pass (torch.utils.checkpoint): the second forward must draw the first one's mask, so ``step`` has to
    be a tensor that is moved on after the backward pass (a number has moved on by then: refused).  As with any module: no eager graph of its parameters
    may be alive while a backward pass through it is captured."""

    def __init__(self, linear, p, seed, relu=False):
        nn.Module.__init__(self)
        self.in_features, self.out_features = linear.in_features, linear.out_features
        self.weight, self.bias = linear.weight, linear.bias
        self.p, self.seed, self.relu, self.step = float(p), int(seed), bool(relu), 0

    def forward(self, x):
        if not self.training:
            y = F.linear(x, self.weight, self.bias)
            return F.relu(y) if self.relu else y
        y = F.linear(x, self.weight).contiguous()
        bias = self.bias if self.bias is None or self.bias.dtype == y.dtype else self.bias.to(y.dtype)      # (under autocast the product's type)
        return self._drop(y, bias, self.relu)

    def extra_repr(self):
        return "%s, p=%g, seed=%d, relu=%s" % (nn.Linear.extra_repr(self), self.p, self.seed, self.relu)


class Mx4LinearLayer(_Counted, nn.Module):
    """``relu?(linear(x))`` with the weight in MXFP4 and x quantised on the way in; the weight is quantised when the layer first runs on a ROCm device
    (its float copy is given up then: code that reads the layer's ``weight`` does not work on it).  Of a ``LinearDropout`` it keeps the dropout, rate, seed
    and step: in training its output is dropped as before.  A state dict holds the float weight or, of a layer that has run, its four bits; a layer in either
    form takes either."""

    def __init__(self, linear, relu=False):
        super().__init__()
        self.in_features, self.out_features, self.relu = linear.in_features, linear.out_features, bool(relu)
        self.p, self.seed, self.step = (linear.p, linear.seed, linear.step) if isinstance(linear, LinearDropout) else (0.0, 0, 0)
        self.register_buffer("weight", linear.weight.detach().clone())
        self.register_buffer("bias", None if linear.bias is None else linear.bias.detach().clone())
        self.register_buffer("codes", None)
        self.register_buffer("scales", None)

    def held(self):
        """the weight as ``ops.Mx4``"""
        from . import ops
        if self.codes is None:
            self._quantise(ops)
        return ops.Mx4(self.codes, self.scales, (self.out_features, self.in_features))

    def _quantise(self, ops):
        """First use, which may be on any stream and in any thread: on the device's default stream, behind what the caller's has been given (so that the
        four bits belong where a module's tensors do), and finished before another stream sees them or the float weight is given up"""
        with _FIRST_USE:
            if self.codes is not None:           # another thread came first
                return
            weight = self.weight
            if not weight.is_cuda:
                raise RuntimeError("Mx4LinearLayer: libadvengine has no CPU path - move the model and its inputs to the ROCm device")
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("Mx4LinearLayer: run the layer once before capturing it (its weight is quantised on first use)")
            home = torch.cuda.default_stream(weight.device)
            home.wait_stream(torch.cuda.current_stream(weight.device))
            with torch.inference_mode(False), torch.no_grad(), torch.cuda.stream(home):
                q = ops.mx4_quantize(weight.contiguous())
            home.synchronize()
            self.scales = q.scales
            self.codes = q.codes                 # (the one that held() asks for: last but the weight)
            self.weight = None

    def _load_from_state_dict(self, state_dict, prefix, *args):
        weight, codes, scales = [state_dict.get(prefix + k) for k in ("weight", "codes", "scales")]
        if codes is not None and scales is not None and weight is None and self.codes is None:
            shape = ((self.in_features + 255) // 256, self.out_features)
            self.codes, self.scales = [torch.empty(shape + (n,), dtype=torch.uint8, device=self.weight.device) for n in (128, 8)]
            self.weight = None
        elif weight is not None and codes is None and scales is None and self.codes is not None:
            if not self.codes.is_cuda:                                       # (moved to the CPU, where nothing is quantised: as it was before it ran)
                self.weight = torch.empty((self.out_features, self.in_features), dtype=weight.dtype, device=self.codes.device)
                self.codes = self.scales = None
            elif tuple(weight.shape) == (self.out_features, self.in_features):
                from . import ops
                held = weight.detach().to(self.codes.device, weight.dtype if weight.dtype in ops._FLOATS else torch.float32)
                q = ops.mx4_quantize(held.contiguous())                      # into the tensors that are there: a captured graph reads those
                state_dict = {k: v for k, v in state_dict.items() if k != prefix + "weight"}
                state_dict[prefix + "codes"], state_dict[prefix + "scales"] = q.codes, q.scales
        super()._load_from_state_dict(state_dict, prefix, *args)

    def forward(self, x):
        w = self.held()
        from . import ops
        bias = self.bias if self.bias is None or self.bias.dtype == x.dtype else self.bias.to(x.dtype)
        y = ops.Mx4Linear.apply(x.contiguous(), w, bias, self.relu)
        return self._drop(y) if self.training and self.p else y        # (behind the ReLU as in front of it: the same values)

    def extra_repr(self):
        return "%d -> %d, mxfp4%s%s" % (self.in_features, self.out_features, ", relu" if self.relu else "", ", p=%g, seed=%d" % (self.p, self.seed) if self.p else "")


class Covering:
    """A convolution whose kernel covers its whole map is a fully connected layer over the map's values (a detector's RoI head: 7x7 on the pooled grid, 1x1
    behind it); whether it does shows when it runs.  Holds such a layer's weight in four bits, beside the float one of the module that asks."""

    def __init__(self):
        self.layer = self.weight = self.stamp = None

    def __call__(self, x, weight, bias, relu):
        """``relu?(x . weight + bias)`` [B, N] of ``x`` [B, C, kh, kw] under ``weight`` [N, C, kh, kw], which is quantised again where it was changed"""
        from . import ops
        # (in-place writes count the version up, ``weight.data = other`` - what ``module.to`` does - moves the pointer)
        stamp = (weight.data_ptr(), weight.device, weight.dtype, None if weight.is_inference() else weight._version)
        if self.weight is not weight or self.stamp != stamp:
            flat = weight.detach().flatten(1)
            if self.layer is not None and self.layer.codes is not None and self.layer.codes.device == weight.device:
                self.layer.load_state_dict({"weight": flat})             # (into the tensors that are there: a captured graph reads those)
            else:
                self.layer = Mx4LinearLayer(types.SimpleNamespace(in_features=flat.shape[1], out_features=flat.shape[0], weight=flat, bias=None))
            self.weight, self.stamp = weight, stamp
        bias = bias if bias is None or bias.dtype == x.dtype else bias.to(x.dtype)
        return ops.Mx4Linear.apply(x.flatten(1).contiguous(), self.layer.held(), bias, bool(relu))


def covers(x, weight, padding, dilation, groups):
    """does the kernel of ``weight`` cover the whole map of ``x``, every value once?"""
    return groups == 1 and x.shape[2:] == weight.shape[2:] and not any(padding) and (weight[0, 0].numel() == 1 or all(d == 1 for d in dilation))


def _is_relu(m):
    """a ReLU that a layer in front of it may take over (one with hooks keeps its place: they want its own result)"""
    return (isinstance(m, nn.ReLU) or type(m).__name__ == "_ReLU") and not _hooked(m)


def _hooked(m):
    return bool(m._forward_hooks or m._forward_pre_hooks or m._backward_hooks or m._backward_pre_hooks)


def _refuse_hooks(who, name, m):
    """Hooks see a layer's own input and result, or make its weight (torch.nn.utils.weight_norm: trained through two other parameters): neither goes over
    to what takes the layer's place"""
    if _hooked(m):
        raise ValueError("%s: %s (%s) has hooks, which its replacement would not run: remove them first" % (who, name, type(m).__name__))


def counter_dropout(module, seed):
    """Replace, IN PLACE, every ``Linear, Dropout(, ReLU)`` run of consecutive children of an ``nn.Sequential`` in ``module`` by ``LinearDropout`` and
    identities - the places in the sequence, hence the state-dict keys, stay.  A ``LinearDropout`` that is there already goes over to ``seed``: from step 0,
    or, where it has run under that seed before, on from its own step.  -> the number of dropout layers that now draw under ``seed``."""
    for parent_name, parent in module.named_modules():                   # (before anything is replaced)
        children = list(parent._modules.items())
        for (name, lin), (drop_name, drop) in zip(children, children[1:]):
            if isinstance(parent, nn.Sequential) and type(lin) is nn.Linear and type(drop) is nn.Dropout:
                _refuse_hooks("counter_dropout", (parent_name + "." if parent_name else "") + name, lin)
                _refuse_hooks("counter_dropout", (parent_name + "." if parent_name else "") + drop_name, drop)
    count = 0
    for parent in list(module.modules()):
        names = list(parent._modules)
        for i, name in enumerate(names):
            lin = parent._modules[name]
            if type(lin) is LinearDropout:
                own = layer_seed(seed, count)
                if lin.seed != own:
                    lin.seed = own
                    if not isinstance(lin.step, torch.Tensor):           # (a step tensor is the program's to move)
                        lin.step = 0
                count += 1
                continue
            drop = parent._modules[names[i + 1]] if isinstance(parent, nn.Sequential) and i + 1 < len(names) else None
            if type(lin) is not nn.Linear or type(drop) is not nn.Dropout:
                continue
            relu = i + 2 < len(names) and _is_relu(parent._modules[names[i + 2]])
            parent._modules[name] = LinearDropout(lin, drop.p, layer_seed(seed, count), relu).train(lin.training)
            parent._modules[names[i + 1]] = nn.Identity().train(lin.training)
            if relu:
                parent._modules[names[i + 2]] = nn.Identity().train(lin.training)
            count += 1
    return count


def _counted(module):
    return {name: m for name, m in module.named_modules() if isinstance(m, LinearDropout) or (isinstance(m, Mx4LinearLayer) and m.p)}


def dropout_state(module):
    """{qualified name: {"seed", "step"}} of the counter-based dropouts under ``module``, plain numbers: what a checkpoint keeps beside the state dict"""
    return {name: {"seed": m.seed, "step": int(m.step)} for name, m in _counted(module).items()}


def load_dropout_state(module, state):
    """The counter-based dropouts under ``module`` go on from where those of ``state`` (``dropout_state``) stood; the two must name the same layers."""
    layers = _counted(module)
    if sorted(layers) != sorted(state):
        raise ValueError("load_dropout_state: the module's dropouts (%s) are not the state's (%s)" % (", ".join(sorted(layers)), ", ".join(sorted(state))))
    for name, m in layers.items():
        m.seed = int(state[name]["seed"])
        if isinstance(m.step, torch.Tensor):
            m.step.fill_(state[name]["step"])
        else:
            m.step = int(state[name]["step"])


def mx4_linears(module, prefix="", fuse_relu=True):
    """Replace, IN PLACE, every ``nn.Linear`` and ``LinearDropout`` under ``module`` by ``Mx4LinearLayer`` (``fuse_relu``: a ReLU that follows it in an
    ``nn.Sequential``, a Dropout between them allowed, runs in its kernel: a dropped or scaled value keeps its sign).  Other subclasses of ``nn.Linear``
    stay (``float_linears`` names them).  -> [(qualified name, what)]"""
    if type(module) in (nn.Linear, LinearDropout):
        raise ValueError("mx4_linears: a layer cannot be replaced in place without the module that holds it: build a heads.Mx4LinearLayer of it")
    refuse_hooked_linears(module, prefix)
    done = []
    for parent_name, parent in list(module.named_modules()):
        names = list(parent._modules)
        for i, name in enumerate(names):
            lin = parent._modules[name]
            if type(lin) not in (nn.Linear, LinearDropout):
                continue
            at = i + 1
            if isinstance(parent, nn.Sequential):
                while at < len(names) and type(parent._modules[names[at]]) in (nn.Dropout, nn.Identity) and not _hooked(parent._modules[names[at]]):
                    at += 1
            follows = fuse_relu and isinstance(parent, nn.Sequential) and at < len(names) and _is_relu(parent._modules[names[at]])
            relu = follows or (type(lin) is LinearDropout and lin.relu)
            parent._modules[name] = Mx4LinearLayer(lin, relu).train(lin.training)
            if follows:
                parent._modules[names[at]] = nn.Identity().train(lin.training)
            done.append((prefix + (parent_name + "." if parent_name else "") + name, "linear %d->%d mxfp4%s" % (lin.in_features, lin.out_features, " + relu" if relu else "")))
    return done


def refuse_hooked_linears(module, prefix=""):
    """raises if a layer that ``mx4_linears`` would replace has hooks"""
    for name, m in module.named_modules():
        if type(m) in (nn.Linear, LinearDropout):
            _refuse_hooks("mx4_linears", prefix + name, m)


def float_linears(module, prefix=""):
    """[(qualified name, type's name)] of the layers under ``module`` (itself included) whose product is still ``nn.Linear``'s or a subclass's"""
    return [(prefix + name, type(m).__name__) for name, m in module.named_modules() if isinstance(m, nn.Linear)]
