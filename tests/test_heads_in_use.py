"""The fully connected heads' layers (heads.py) in the hands of a program that does more than call them once: recomputed activations, a second seed, a
head that was trained before it is quantised, checkpoints, hooks, a first call on a side stream.  Without a GPU the oracle stands in the kernel's place."""
import numpy as np
import pytest
import torch
import torch.nn as nn
from torch.utils.checkpoint import checkpoint

from eval_driving_safety_amd import heads
from oracle import oracle_np as O


class OracleDropout(torch.autograd.Function):
    """``ops.Dropout`` on the CPU, from the oracle"""

    @staticmethod
    def forward(ctx, x, p, seed, step=0, bias=None, relu=False):
        y = torch.tensor(O.dropout(x.detach().double().numpy(), p, seed, int(step), None if bias is None else bias.detach().double().numpy(), relu)).to(x.dtype)
        ctx.save_for_backward(y if relu else None, step if isinstance(step, torch.Tensor) else None)
        ctx.p, ctx.seed, ctx.step = p, seed, int(step)
        return y

    @staticmethod
    def backward(ctx, g):
        y, step = ctx.saved_tensors
        gx, gb = O.dropout_bwd(g.double().numpy(), ctx.p, ctx.seed, ctx.step if step is None else int(step), None if y is None else y.double().numpy())
        return torch.tensor(gx).to(g.dtype), None, None, None, torch.tensor(gb).to(g.dtype) if ctx.needs_input_grad[4] else None, None


@pytest.fixture
def on_the_cpu(monkeypatch):
    from eval_driving_safety_amd import ops
    monkeypatch.setattr(ops, "Dropout", OracleDropout)


def small_head(seed=0, p=0.5):
    torch.manual_seed(seed)
    return nn.Sequential(nn.Linear(24, 40), nn.Dropout(p), nn.ReLU(), nn.Linear(40, 3), nn.Dropout(p))


def rows(n, seed=1):
    return torch.randn(n, 24, generator=torch.Generator().manual_seed(seed))


# ---------------------------------------------------------------------------------------------------------------- recomputed activations
def recomputed_gradient(device, use_reentrant, step):
    """(output, gradient w.r.t. the input) of a LinearDropout, and of the same one under activation recomputation"""
    out = []
    for recompute in (False, True):
        h = small_head().to(device)
        heads.counter_dropout(h, 5)
        layer = h[0].train()
        layer.step = step if isinstance(step, int) else step.clone()
        x = rows(6).to(device).requires_grad_()
        y = checkpoint(layer, x, use_reentrant=use_reentrant) if recompute else layer(x)
        y.sum().backward()
        out.append((y.detach(), x.grad))
    return out


def check_recomputation(device):
    for use_reentrant in (False, True):
        with pytest.raises(RuntimeError, match="recompute"):
            recomputed_gradient(device, use_reentrant, 3)
        (y, g), (yr, gr) = recomputed_gradient(device, use_reentrant, torch.full((1,), 3, dtype=torch.int64, device=device))
        assert torch.equal(y, yr) and torch.equal(g, gr) and g.abs().max() > 0


def test_a_recomputed_forward_is_refused_or_draws_the_same_mask(on_the_cpu):
    """a numbered step has moved on when the forward runs again inside the backward pass: another mask than the loss saw - refused; a step tensor holds"""
    check_recomputation(torch.device("cpu"))


@pytest.mark.gpu
def test_hip_a_recomputed_forward_is_refused_or_draws_the_same_mask():
    check_recomputation(torch.device("cuda"))


# ---------------------------------------------------------------------------------------------------------------- first use
@pytest.mark.gpu
def test_hip_the_first_call_may_be_on_a_side_stream_and_the_second_on_another():
    """the weight is quantised inside the first forward: a second stream's forward must find it finished, and memory handed out again on the stream that
    made the float weight must not be read any more"""
    import threading
    from eval_driving_safety_amd import ops
    torch.manual_seed(2)
    lin = nn.Linear(4096, 2048).cuda()
    x = torch.randn(9, 4096, generator=torch.Generator().manual_seed(2)).cuda()
    want = ops.mx4_linear(x, ops.mx4_quantize(lin.weight.detach()), lin.bias.detach())
    for threads in (False, True):
        layer = nn.Sequential(heads.Mx4LinearLayer(lin))
        torch.cuda.synchronize()
        a, b = torch.cuda.Stream(), torch.cuda.Stream()
        got = {}

        def call(stream, name, wait):
            with torch.no_grad(), torch.cuda.stream(stream):
                if wait:
                    torch.cuda._sleep(2_000_000)              # work in front of the first use
                got[name] = layer(x)

        if threads:
            both = [threading.Thread(target=call, args=(s, n, True)) for s, n in ((a, "a"), (b, "b"))]
            for t in both:
                t.start()
            for t in both:
                t.join()
        else:
            call(a, "a", True)
            spoil = [torch.full((2048, 4096), float("nan"), device="cuda") for _ in range(3)]      # the size of what the layer gave up
            call(b, "b", False)
            del spoil
        torch.cuda.synchronize()
        assert torch.equal(got["a"], want) and torch.equal(got["b"], want) and layer[0].weight is None


@pytest.mark.gpu
def test_hip_a_layer_first_run_in_inference_mode_carries_gradients_afterwards():
    from eval_driving_safety_amd import ops
    torch.manual_seed(3)
    lin = nn.Linear(24, 8).cuda()
    layer = heads.Mx4LinearLayer(lin)
    x = rows(5).cuda()
    with torch.inference_mode():
        y = layer(x)
    xr = x.clone().requires_grad_()
    z = layer(xr)
    z.sum().backward()
    assert torch.equal(y, z) and torch.equal(xr.grad, ops.mx4_linear_dgrad(torch.ones_like(z), layer.held()))


# ---------------------------------------------------------------------------------------------------------------- trained, then quantised
def test_a_head_trained_under_counter_dropout_is_quantised(on_the_cpu):
    h = small_head()
    heads.counter_dropout(h, 5)
    h.train()
    h(rows(2))
    counted = [m for m in h if isinstance(m, heads.LinearDropout)]
    done = heads.mx4_linears(h)
    assert [n for n, _ in done] == ["0", "3"] and [w for _, w in done] == ["linear 24->40 mxfp4 + relu", "linear 40->3 mxfp4"]
    held = [m for m in h if isinstance(m, heads.Mx4LinearLayer)]
    assert [(m.relu, m.p, m.seed, m.step, m.training) for m in held] == [(m.relu, m.p, m.seed, 1, True) for m in counted]
    for m, c in zip(held, counted):
        assert torch.equal(m.weight, c.weight) and torch.equal(m.bias, c.bias) and not m.weight.requires_grad


def test_adopt_quantises_a_head_trained_under_counter_dropout():
    from eval_driving_safety_amd import adopt as A
    h = nn.Sequential(small_head())
    heads.counter_dropout(h, 5)
    report = A.adopt(h.eval(), linear="mxfp4", functional=False)
    assert [n for n, _ in report["replaced"]] == ["0.0", "0.3"]


@pytest.mark.gpu
def test_hip_train_then_quantise_then_validate(tmp_path):
    """classifiers.train under a dropout seed, quantize_head, check_accuracy: the accuracy is that of the four-bit layers; in training the dropout is the
    one the layer had"""
    from eval_driving_safety_amd import classifiers as C, ops

    class Tiny(nn.Module):
        head_key = "classifier"

        def __init__(self):
            super().__init__()
            torch.manual_seed(4)
            self.net = nn.Module()
            self.net.classifier = nn.Sequential(nn.Linear(24, 40), nn.Dropout(0.1), nn.ReLU(), nn.Linear(40, 1), nn.Dropout(0.1), nn.Sigmoid())

        backbone = property(lambda self: self.net)

        def forward(self, x):
            return self.net.classifier(x).squeeze(1)

    data = [(rows(16, 7 + k), (rows(16, 7 + k)[:, 0] > 0).float()) for k in range(4)]
    m = C.train("driving_constraint", data, None, torch.device("cuda"), str(tmp_path), epochs=2, model=Tiny(), log=lambda *a: None, dropout_seed=7)
    head = m.net.classifier
    (w1, b1), (w2, b2) = [(ops.mx4_quantize(q.weight.detach()), q.bias.detach()) for q in head if isinstance(q, heads.LinearDropout)]
    assert [n for n, _ in C.quantize_head(m)] == ["classifier.0", "classifier.3"]
    acc = C.check_accuracy(data, m, torch.device("cuda"), log=lambda *a: None)
    right = sum(int(((torch.sigmoid(ops.mx4_linear(ops.mx4_linear(x.cuda(), w1, b1, True), w2, b2))[:, 0] >= 0.5) == (t.cuda() > 0)).sum()) for x, t in data)
    assert acc == right / 64 * 100
    layer, x = head[0], data[0][0].cuda()
    assert layer.training and layer.p == 0.1 and layer.step == 8                  # as check_accuracy leaves the model; two epochs of four batches
    plain = layer.eval()(x)
    dropped = layer.train()(x)
    kept = O.dropout_kept(0, 16 * 40, 0.1, layer.seed, 8).reshape(16, 40)
    np.testing.assert_allclose(dropped.detach().cpu().numpy(), np.where(kept, plain.cpu().numpy() / 0.9, 0), rtol=3 * 2.0 ** -23, atol=0)
    assert layer.step == 9


# ---------------------------------------------------------------------------------------------------------------- another seed
def test_a_second_seed_takes_the_place_of_the_first(on_the_cpu):
    h, fresh = small_head(), small_head()
    assert heads.counter_dropout(h, 7) == 2
    h.train()
    h(rows(2)), h(rows(2))
    assert heads.counter_dropout(h, 8) == 2 and heads.counter_dropout(fresh, 8) == 2
    layers, new = [[m for m in q if isinstance(m, heads.LinearDropout)] for q in (h, fresh)]
    assert [(m.seed, m.step) for m in layers] == [(m.seed, 0) for m in new]
    assert torch.equal(h(rows(4)), fresh.train()(rows(4)))                       # as a model that never had another
    assert heads.counter_dropout(h, 8) == 2 and [m.step for m in layers] == [1, 1]        # the same seed again: its masks are not repeated
    layers[0].step = torch.tensor([5])
    assert heads.counter_dropout(nn.ModuleDict({"a": layers[0]}), 3) == 1 and int(layers[0].step) == 5 and layers[0].seed == heads.layer_seed(3, 0)


# ---------------------------------------------------------------------------------------------------------------- nothing to replace
def holder(head):
    class Model(nn.Module):
        head_key = "fc"

        def __init__(self):
            super().__init__()
            self.net = nn.Module()
            self.net.fc = head

        backbone = property(lambda self: self.net)

        def forward(self, x):
            return self.net.fc(x).squeeze(1)

    return Model()


class OwnLinear(nn.Linear):
    pass


def test_a_head_of_which_nothing_can_be_replaced_is_refused(tmp_path):
    from eval_driving_safety_amd import adopt as A, classifiers as C
    with pytest.raises(ValueError, match="no Linear layer"):
        C.quantize_head(holder(nn.Sequential(nn.Sigmoid())))
    with pytest.raises(ValueError, match="fc.1 .OwnLinear."):
        C.quantize_head(holder(nn.Sequential(nn.Linear(4, 4), OwnLinear(4, 1))))
    with pytest.raises(ValueError, match="cannot be replaced in place"):
        heads.mx4_linears(nn.Linear(4, 4))
    with pytest.raises(ValueError, match="cannot be adopted"):
        A.adopt(nn.Linear(4, 4).eval(), linear="mxfp4", functional=False)
    report = A.adopt(nn.Sequential(nn.Linear(4, 4), OwnLinear(4, 1)).eval(), linear="mxfp4", functional=False)
    assert [n for n, _ in report["replaced"]] == ["0"] and [n for n, _ in report["kept"]] == ["1"]
    m = holder(nn.Linear(4, 1))                                                   # a head that is one layer
    assert C.quantize_head(m) == [("fc", "linear 4->1 mxfp4")] and isinstance(m.net.fc, heads.Mx4LinearLayer)
    m = holder(nn.Sequential(nn.Linear(4, 1)))
    assert len(C.quantize_head(m)) == 1 and C.quantize_head(m) == []              # nothing left to do
    for head in (nn.Sequential(nn.Linear(4, 1), nn.Sigmoid()), nn.Linear(4, 1)):
        with pytest.raises(ValueError, match="dropout_seed"):
            C.train("driving_constraint", [], None, torch.device("cpu"), str(tmp_path), epochs=1, model=holder(head), log=lambda *a: None, dropout_seed=1)


def test_adopt_leaves_relus_alone_where_it_is_told_to():
    from eval_driving_safety_amd import adopt as A
    for fuse in (True, False):
        h = small_head().eval()
        A.adopt(h, fuse_relu=fuse, linear="mxfp4", functional=False)
        assert h[0].relu is fuse and isinstance(h[2], nn.Identity if fuse else nn.ReLU)


# ---------------------------------------------------------------------------------------------------------------- hooks
def test_hooked_layers_are_refused_and_hooked_relus_keep_their_place():
    import warnings
    from eval_driving_safety_amd import adopt as A
    hooks = (lambda m: m.register_forward_hook(lambda *a: None), lambda m: m.register_forward_pre_hook(lambda *a: None),
             lambda m: m.register_full_backward_hook(lambda *a: None), lambda m: m.register_full_backward_pre_hook(lambda *a: None))
    for add in hooks:
        for replace in (lambda q: heads.counter_dropout(q, 1), heads.mx4_linears, lambda q: A.adopt(q.eval(), linear="mxfp4", functional=False)):
            h = nn.Sequential(nn.Conv2d(1, 1, 1), nn.ReLU(), small_head())
            add(h[2][3])
            kinds = [type(m) for m in h.modules()]
            with pytest.raises(ValueError, match="2.3 .Linear. has hooks"):
                replace(h)
            assert [type(m) for m in h.modules()] == kinds                          # nothing was replaced
        h = small_head()
        add(h[1])
        with pytest.raises(ValueError, match="1 .Dropout. has hooks"):
            heads.counter_dropout(h, 1)
        heads.mx4_linears(h)
        assert not h[0].relu and isinstance(h[2], nn.ReLU)                          # its hook sees what it saw
        for replace in (lambda q: heads.counter_dropout(q, 1), heads.mx4_linears):
            h = small_head()
            add(h[2])
            replace(h)
            assert not h[0].relu and isinstance(h[2], nn.ReLU)
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        h = nn.Sequential(nn.utils.weight_norm(nn.Linear(4, 4)), nn.Dropout(0.1))      # its weight is made by a hook, of two other parameters
    with pytest.raises(ValueError, match="hooks"):
        heads.counter_dropout(h, 1)


def test_a_dropout_that_would_still_draw_from_the_process_is_refused(tmp_path):
    from eval_driving_safety_amd import classifiers as C
    head = nn.Sequential(nn.Linear(4, 4), nn.Dropout(0.1), nn.Linear(4, 4), nn.ReLU(), nn.Dropout(0.2), nn.Linear(4, 1))
    with pytest.raises(ValueError, match="fc.4 does not follow a Linear"):
        C.train("driving_constraint", [], None, torch.device("cpu"), str(tmp_path), epochs=1, model=holder(head), log=lambda *a: None, dropout_seed=1)


# ---------------------------------------------------------------------------------------------------------------- state dicts
def four_bit_layer(lin, codes):
    """a Mx4LinearLayer as it is after its first run"""
    layer = heads.Mx4LinearLayer(lin)
    layer.codes, layer.scales, layer.weight = torch.randint(0, 256, codes, dtype=torch.uint8), torch.randint(100, 150, codes[:2] + (8,), dtype=torch.uint8), None
    return layer


def test_a_layer_in_either_form_takes_either_state():
    used, lin = four_bit_layer(nn.Linear(300, 5), (2, 5, 128)), nn.Linear(300, 5)
    fresh = heads.Mx4LinearLayer(nn.Linear(300, 5))
    fresh.load_state_dict(used.state_dict())
    assert fresh.weight is None and torch.equal(fresh.codes, used.codes) and torch.equal(fresh.scales, used.scales) and torch.equal(fresh.bias, used.bias)
    again = four_bit_layer(nn.Linear(300, 5), (2, 5, 128))
    again.load_state_dict(used.state_dict())
    assert torch.equal(again.codes, used.codes)
    for strict in (True, False):
        used.load_state_dict(lin.state_dict(), strict=strict)                       # on the CPU: float until it runs on a device
        assert used.codes is None and used.scales is None and torch.equal(used.weight, lin.weight) and torch.equal(used.bias, lin.bias)
        used = four_bit_layer(nn.Linear(300, 5), (2, 5, 128))
    net, state = nn.Sequential(nn.ReLU(), heads.Mx4LinearLayer(nn.Linear(300, 5))), nn.Sequential(nn.ReLU(), used).state_dict()
    net.load_state_dict(state)
    assert torch.equal(net[1].codes, used.codes)
    for bad in (nn.Linear(299, 5), nn.Linear(300, 6)):
        for layer in (used, heads.Mx4LinearLayer(lin)):
            with pytest.raises(RuntimeError):
                layer.load_state_dict(bad.state_dict())
            used = four_bit_layer(nn.Linear(300, 5), (2, 5, 128))
    with pytest.raises(RuntimeError):
        heads.Mx4LinearLayer(nn.Linear(256, 5)).load_state_dict(used.state_dict())
    with pytest.raises(RuntimeError):
        heads.Mx4LinearLayer(lin).load_state_dict({k: v for k, v in used.state_dict().items() if k != "scales"})


@pytest.mark.gpu
def test_hip_float_weights_loaded_into_a_layer_that_has_run():
    """they are quantised into the tensors that are there: the eager call and a graph that was captured before give the new layer's values"""
    from eval_driving_safety_amd import ops
    torch.manual_seed(6)
    a, b = nn.Linear(300, 70).cuda(), nn.Linear(300, 70).cuda()
    x = torch.randn(40, 300, generator=torch.Generator().manual_seed(6)).cuda()
    want = [ops.mx4_linear(x, ops.mx4_quantize(q.weight.detach()), q.bias.detach()) for q in (a, b)]
    layer = heads.Mx4LinearLayer(a)
    with torch.no_grad():
        assert torch.equal(layer(x), want[0])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = layer(x)
        for lin, w in ((b, want[1]), (a, want[0]), (b, want[1])):
            for strict, move in ((True, "cuda"), (False, "cpu")):
                layer.load_state_dict({k: v.to(move) for k, v in lin.state_dict().items()}, strict=strict)
                graph.replay()
                torch.cuda.synchronize()
                assert torch.equal(layer(x), w) and torch.equal(y, w) and layer.weight is None
        fresh = heads.Mx4LinearLayer(a).cuda()
        fresh.load_state_dict(layer.state_dict())
        assert torch.equal(fresh(x), want[1])
        layer.load_state_dict({"weight": b.weight.double(), "bias": b.bias})
        assert torch.equal(layer(x), want[1])
        with pytest.raises(RuntimeError):
            layer.load_state_dict(nn.Linear(299, 70).state_dict())
        # (as any module's: of a state that does not fit, the tensors that do - the bias - are taken before the error)
        assert torch.equal(layer(x), ops.mx4_linear(x, ops.mx4_quantize(b.weight.detach()), layer.bias))


# ---------------------------------------------------------------------------------------------------------------- going on from a checkpoint
def test_training_goes_on_from_a_checkpoint_with_the_masks_that_follow(on_the_cpu, tmp_path):
    from eval_driving_safety_amd import classifiers as C

    def model():
        return holder(nn.Sequential(small_head(8), nn.Linear(3, 1), nn.Dropout(0.1), nn.Sigmoid()))

    def run(m, data, where):
        return C.train("dynamic_vehicles", data, None, torch.device("cpu"), str(tmp_path / where), epochs=1, model=m, log=lambda *a: None, dropout_seed=9)

    data = [(rows(4, k), torch.tensor([0.0, 1.0, 1.0, 0.0])) for k in range(5)]
    m = run(model(), data[:3], "a")
    saved = torch.load(tmp_path / "a" / "cnn_1.pth")
    assert [v["step"] for v in saved["dropout_state"].values()] == [3, 3, 3] and list(saved["model_state_dict"]) == list(model().state_dict())
    on = model()
    heads.counter_dropout(on.net.fc, 9)
    C.load_checkpoint(on, tmp_path / "a" / "cnn_1.pth")
    for q in (m, on):
        run(q, data[3:], "b")
    assert heads.dropout_state(m) == heads.dropout_state(on) and all(v["step"] == 5 for v in heads.dropout_state(on).values())
    assert all(torch.equal(a, b) for a, b in zip(m.state_dict().values(), on.state_dict().values()))
    plain = C.load_checkpoint(model(), tmp_path / "a" / "cnn_1.pth")              # without counter-based layers: the weights alone
    assert heads.dropout_state(plain) == {}
    C.train("dynamic_vehicles", data[:1], None, torch.device("cpu"), str(tmp_path / "c"), epochs=1, model=plain, log=lambda *a: None)
    assert "dropout_state" not in torch.load(tmp_path / "c" / "cnn_1.pth")
    layer = on.net.fc[0][0]
    layer.step = torch.zeros(1, dtype=torch.int64)
    C.load_checkpoint(on, tmp_path / "a" / "cnn_1.pth")
    assert int(layer.step) == 3
    with pytest.raises(ValueError, match="not the state's"):
        heads.load_dropout_state(on, {"fc": {"seed": 1, "step": 1}})


def test_the_command_refuses_options_of_the_other_mode(capsys):
    from eval_driving_safety_amd.cli import classifier
    for argv, word in ((["dynamic_vehicles", "validate", "--dropout_seed", "7"], "--dropout_seed"), (["driving_constraint", "train", "--head", "mxfp4"], "--head")):
        with pytest.raises(SystemExit) as e:
            classifier.main(argv)
        assert e.value.code == 2 and word + " " in capsys.readouterr().err


# ---------------------------------------------------------------------------------------------------------------- weights between the passes
def test_a_weight_changed_between_the_passes_is_refused(monkeypatch):
    from eval_driving_safety_amd import ops
    from eval_driving_safety_amd.ops import mx4
    monkeypatch.setattr(mx4, "mx4_linear", lambda x, w, bias, relu: x.detach()[:, :w.rows].clone())
    monkeypatch.setattr(mx4, "mx4_linear_dgrad", lambda g, w, mask: torch.nn.functional.pad(g, (0, w.cols - w.rows)))
    for inference in (False, True):
        with torch.inference_mode(inference):
            w = ops.Mx4(torch.zeros((1, 5, 128), dtype=torch.uint8), torch.zeros((1, 5, 8), dtype=torch.uint8), (5, 24))
        x = rows(3).requires_grad_()
        ops.Mx4Linear.apply(x, w).sum().backward()
        assert bool((x.grad[:, :5] == 1).all()) and not x.grad[:, 5:].any()
    for name in ("codes", "scales"):
        w = ops.Mx4(torch.zeros((1, 5, 128), dtype=torch.uint8), torch.zeros((1, 5, 8), dtype=torch.uint8), (5, 24))
        y = ops.Mx4Linear.apply(x, w)
        getattr(w, name).add_(1)
        with pytest.raises(RuntimeError, match="changed in place"):
            y.sum().backward()


# ---------------------------------------------------------------------------------------------------------------- arguments left out
def test_autograd_functions_with_the_arguments_left_out_that_may_be(monkeypatch):
    from eval_driving_safety_amd import ops
    import sys
    dropout, mx4 = sys.modules["eval_driving_safety_amd.ops.dropout"], sys.modules["eval_driving_safety_amd.ops.mx4"]
    monkeypatch.setattr(dropout, "dropout", lambda x, p, seed, step, bias, relu: torch.tensor(O.dropout(x.detach().numpy(), p, seed, step)).float())
    monkeypatch.setattr(dropout, "dropout_bwd", lambda g, p, seed, step, y, with_bias: (torch.tensor(O.dropout_bwd(g.numpy(), p, seed, step)[0]).float(), None))
    for extra in ((), (3,), (3, None), (3, None, False)):
        x = rows(4).requires_grad_()
        ops.Dropout.apply(x, 0.5, 7, *extra).sum().backward()
        kept = O.dropout_kept(0, 96, 0.5, 7, 3 if extra else 0).reshape(4, 24)
        assert np.array_equal(x.grad.numpy(), kept * 2.0)
    monkeypatch.setattr(mx4, "mx4_linear", lambda x, w, bias, relu: x.detach()[:, :w.rows].clone())
    monkeypatch.setattr(mx4, "mx4_linear_dgrad", lambda g, w, mask: torch.nn.functional.pad(g, (0, w.cols - w.rows)))
    w = ops.Mx4(torch.zeros((1, 5, 128), dtype=torch.uint8), torch.zeros((1, 5, 8), dtype=torch.uint8), (5, 24))
    for extra in ((), (None,), (None, False), (torch.zeros(5),)):
        x = rows(3).requires_grad_()
        ops.Mx4Linear.apply(x, w, *extra).sum().backward()
        assert bool((x.grad[:, :5] == 1).all()) and not x.grad[:, 5:].any()
    with pytest.raises(ValueError):
        ops.Mx4Linear.apply(rows(3), w, torch.zeros(5, requires_grad=True))


@pytest.mark.gpu
def test_hip_autograd_functions_with_the_arguments_left_out_that_may_be():
    from eval_driving_safety_amd import ops
    x = rows(4).cuda().requires_grad_()
    g, = torch.autograd.grad(ops.Dropout.apply(x, 0.5, 7).sum(), x)
    assert torch.equal(g, ops.dropout_bwd(torch.ones_like(x), 0.5, 7)[0])
    w = ops.mx4_quantize(rows(5, 2).cuda())
    g, = torch.autograd.grad(ops.Mx4Linear.apply(x, w).sum(), x)
    assert torch.equal(g, ops.mx4_linear_dgrad(torch.ones((4, 5), device="cuda"), w))
    w.codes.zero_()
    y = ops.Mx4Linear.apply(x, w)
    w.scales.add_(1)
    with pytest.raises(RuntimeError, match="changed in place"):
        y.sum().backward()


# ---------------------------------------------------------------------------------------------------------------- captured training
@pytest.mark.gpu
def test_hip_a_captured_forward_and_backward_draw_as_the_step_moves_on():
    """a step of the layer and its gradients in one graph, replayed with the program's eager work between; then under activation recomputation, captured too"""
    h = small_head(9).cuda()
    heads.counter_dropout(h, 11)
    layer = h[0].train()
    layer.step = torch.zeros((1,), dtype=torch.int64, device="cuda")
    x = rows(33, 5).cuda().requires_grad_()
    g = torch.randn(33, 40, generator=torch.Generator().manual_seed(5)).cuda()

    def step(recompute):
        y = checkpoint(layer, x, use_reentrant=False, preserve_rng_state=False) if recompute else layer(x)
        return (y.detach(),) + torch.autograd.grad(y, (x, layer.weight, layer.bias), g)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for recompute in (False, True):
            step(recompute)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for recompute in (False, True):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(recompute)
        graphs.append((graph, out))
    seen = []
    for k in (4, 9, 4, 6):
        layer.step.fill_(k)
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        eager = step(False)
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, eager)), k
        kept = O.dropout_kept(0, 33 * 40, 0.5, layer.seed, k).reshape(33, 40)
        assert not eager[0].cpu().numpy()[~kept].any()
        seen.append(eager[1].clone())
    assert torch.equal(seen[0], seen[2]) and not torch.equal(seen[0], seen[1])


# ---------------------------------------------------------------------------------------------------------------- convolutions that are fully connected
def test_which_convolutions_cover_their_map():
    x = torch.zeros(2, 3, 7, 5)
    yes = lambda w, p=(0, 0), d=(1, 1), g=1, m=x: heads.covers(m, torch.zeros(w), p, d, g)      # noqa: E731
    assert yes((4, 3, 7, 5)) and yes((4, 3, 1, 1), d=(2, 2), m=torch.zeros(2, 3, 1, 1))
    assert not yes((4, 3, 7, 7)) and not yes((4, 3, 7, 5), p=(1, 1)) and not yes((4, 3, 7, 5), d=(2, 2)) and not yes((3, 1, 7, 5), g=3)
    assert not yes((4, 3, 1, 1))


@pytest.mark.gpu
def test_hip_an_adopted_roi_heads_fully_connected_convolutions_are_in_four_bits():
    """7x7 convolution on the pooled grid - ReLU - 1x1 - ReLU, as a Stereo R-CNN head has them: each layer the four-bit product of its own input, the
    gradient straight through; on another map the same layer keeps its float convolution"""
    from eval_driving_safety_amd import adopt as A, ops
    torch.manual_seed(10)
    net = nn.Sequential(nn.Conv2d(8, 48, 7, stride=7), nn.ReLU(), nn.Conv2d(48, 40, 1), nn.ReLU()).eval().cuda()
    w = [net[0].weight.detach().flatten(1).clone(), net[2].weight.detach().flatten(1).clone()]
    b = [net[0].bias.detach().clone(), net[2].bias.detach().clone()]
    plain = [p.detach().clone() for p in (net[0].weight, net[0].bias)]
    A.adopt(net, linear="mxfp4", functional=False)
    assert [(n, m.relu) for n, m in net.named_children() if isinstance(m, A.AdoptedConv2d)] == [("0", True), ("2", True)]
    x = torch.randn(33, 8, 7, 7, generator=torch.Generator().manual_seed(10)).cuda().requires_grad_()
    y = net(x)
    q = [ops.mx4_quantize(v) for v in w]
    z1 = ops.mx4_linear(x.detach().flatten(1), q[0], b[0], True)
    z2 = ops.mx4_linear(z1, q[1], b[1], True)
    assert y.shape == (33, 40, 1, 1) and torch.equal(y.flatten(1), z2)
    g = torch.randn(33, 40, generator=torch.Generator().manual_seed(11)).cuda()
    y.backward(g[:, :, None, None])
    gx = ops.mx4_linear_dgrad(ops.mx4_linear_dgrad(g, q[1], z2), q[0], z1)
    assert torch.equal(x.grad.flatten(1), gx) and gx.abs().max() > 0
    far = torch.randn(2, 8, 14, 7, generator=torch.Generator().manual_seed(12)).cuda()
    with torch.no_grad():
        want = torch.relu(nn.functional.conv2d(far.double(), plain[0].double(), plain[1].double(), stride=7))
        # 392 float32 products and additions a value
        assert bool(((net[0](far).double() - want).abs() <= 400 * 2.0 ** -23 * nn.functional.conv2d(far.double().abs(), plain[0].double().abs(), plain[1].double().abs(), stride=7)).all())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = net(x)
        net[0].weight.mul_(2)                                                 # quantised again, into what the captured graph reads
        z1 = ops.mx4_linear(x.detach().flatten(1), ops.mx4_quantize(2 * w[0]), b[0], True)
        want = ops.mx4_linear(z1, q[1], b[1], True)
        for _ in range(3):
            assert torch.equal(net(x).flatten(1), want)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out.flatten(1), want)


@pytest.mark.gpu
def test_hip_the_surrogate_detectors_roi_head_in_four_bits():
    from eval_driving_safety_amd import adopt as A, ops
    from eval_driving_safety_amd.surrogates import StereoRcnnR101
    net = StereoRcnnR101(blocks=(1, 1, 1, 1), rois_per_image=16).eval().cuda()
    pooled = torch.relu(torch.randn(37, 512, 7, 7, generator=torch.Generator().manual_seed(13))).cuda().requires_grad_()
    float_top = net.head_to_tail(pooled).detach()
    A.adopt(net, linear="mxfp4", functional=False)
    top = net.head_to_tail(pooled)
    q7, q1 = [ops.mx4_quantize(m.weight.flatten(1).contiguous()) for m in (net.top7, net.top1)]
    z7 = ops.mx4_linear(pooled.detach().flatten(1), q7, net.top7.bias, True)
    z1 = ops.mx4_linear(z7, q1, net.top1.bias, True)
    assert torch.equal(top, z1) and not torch.equal(top, float_top)
    g = torch.randn(37, 2048, generator=torch.Generator().manual_seed(14)).cuda()
    got, = torch.autograd.grad(top, pooled, g)
    assert torch.equal(got.flatten(1), ops.mx4_linear_dgrad(ops.mx4_linear_dgrad(g, q1, z1), q7, z7))
    assert isinstance(net.cls_score, heads.Mx4LinearLayer)


@pytest.mark.gpu
@pytest.mark.parametrize("boxes", [0, 1, 5])
def test_hip_covering_layers_on_slices_of_maps_and_without_boxes(boxes):
    from eval_driving_safety_amd import adopt as A
    torch.manual_seed(15)
    net = nn.Sequential(nn.Conv2d(8, 6, 1), nn.ReLU()).eval().cuda()
    A.adopt(net, linear="mxfp4", functional=False)
    whole = torch.randn(boxes, 16, 1, 1, generator=torch.Generator().manual_seed(15)).cuda()
    for x in (whole[:, :8], whole[:, ::2], whole[:, 8:].contiguous(memory_format=torch.channels_last)):
        xr = x.detach().requires_grad_()
        y = net(xr)
        assert y.shape == (boxes, 6, 1, 1) and torch.equal(y, net(x.clone().contiguous()))
        y.sum().backward()
        assert xr.grad.shape == x.shape


@pytest.mark.gpu
def test_hip_a_covering_layer_follows_its_weight():
    """written in place, given other memory, moved away and back, and to another type"""
    from eval_driving_safety_amd import ops
    gen = torch.Generator().manual_seed(16)
    x = torch.randn(9, 8, 3, 3, generator=gen).cuda()
    m = nn.Conv2d(8, 6, 3).cuda().requires_grad_(False)
    covering = heads.Covering()

    def check(x=x):
        want = ops.mx4_linear(x.flatten(1), ops.mx4_quantize(m.weight.flatten(1)), m.bias, True)
        assert torch.equal(covering(x, m.weight, m.bias, True), want)
        return want

    first = check()
    m.weight.mul_(-1)
    assert not torch.equal(check(), first)
    m.weight.data = torch.randn(6, 8, 3, 3, generator=gen).cuda()
    second = check()
    m.cpu()
    m.weight.mul_(2)
    m.cuda()
    assert not torch.equal(check(), second)
    m.weight = nn.Parameter(torch.randn(6, 8, 3, 3, generator=gen).cuda(), requires_grad=False)
    check()
    m.half()
    check(x.half())
