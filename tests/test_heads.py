"""The fully connected heads on this package's kernels, put together: the classifiers' training step under a counter-based dropout, validation with
four-bit weights, an adopted detector head with four-bit weights under an attack's gradient."""
import numpy as np
import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from eval_driving_safety_amd import adopt as A
from eval_driving_safety_amd import classifiers as C
from eval_driving_safety_amd import heads
from oracle import oracle_np as O


def small_head(seed=0):
    torch.manual_seed(seed)
    return nn.Sequential(C._Flatten(), nn.Linear(72, 40), nn.Dropout(0.1), C._ReLU(), nn.Linear(40, 1), nn.Dropout(0.1), nn.Sigmoid())


def test_counter_dropout_keeps_the_layout():
    m = C.DrivingConstraintCNN()
    keys = list(m.state_dict())
    assert heads.counter_dropout(m.resnet50.fc, 5) == 1 and list(m.state_dict()) == keys
    h = small_head()
    keys, x = list(h.state_dict()), torch.randn(3, 2, 36)
    want = h.eval()(x)
    assert heads.counter_dropout(h, 5) == 2 and list(h.state_dict()) == keys
    lins = [q for q in h if isinstance(q, heads.LinearDropout)]
    assert [q.relu for q in lins] == [True, False] and lins[0].seed != lins[1].seed and isinstance(h[3], nn.Identity)
    assert torch.equal(h(x), want) and not any(q.training for q in h)            # eval: no dropout, the same values
    with pytest.raises(TypeError):
        h.train()(x)                                                             # training has no CPU path


def test_mx4_linears_replaces_and_refuses_the_cpu():
    h = small_head().eval()
    done = heads.mx4_linears(h)
    assert [n for n, _ in done] == ["1", "4"] and h[1].relu and not h[4].relu and isinstance(h[3], nn.Identity)
    with pytest.raises(RuntimeError):
        h(torch.randn(3, 72))
    with pytest.raises(ValueError):
        A.adopt(nn.Sequential(nn.Linear(4, 4)).eval(), linear="int4")
    m = C.DynamicVehicleCNN()
    assert [n for n, _ in C.quantize_head(m)] == ["classifier.1", "classifier.4"]


def test_cli_knows_the_options():
    from eval_driving_safety_amd.cli import classifier
    a = classifier.build_parser().parse_args(["dynamic_vehicles", "train", "--dropout_seed", "7"])
    assert a.dropout_seed == 7 and a.head == "float32"
    assert classifier.build_parser().parse_args(["driving_constraint", "validate", "--head", "mxfp4"]).head == "mxfp4"


# ---------------------------------------------------------------------------------------------------------------- on the GPU
@pytest.mark.gpu
def test_training_step_gradients_against_the_formula():
    """head with dropout in training: output and every gradient against float64 products with the oracle's masks"""
    h = small_head().cuda()
    heads.counter_dropout(h, 99)
    h.train()
    x = torch.randn(5, 72, generator=torch.Generator().manual_seed(1)).cuda().requires_grad_()
    h(x)                                                  # step 0
    y = h(x)                                              # step 1
    loss = F.binary_cross_entropy(y, torch.tensor([[0.0], [1.0], [1.0], [0.0], [1.0]]).cuda())
    loss.backward()
    l1, l2 = h[1], h[4]
    w1, b1, w2, b2 = [p.detach().double().cpu().numpy() for p in (l1.weight, l1.bias, l2.weight, l2.bias)]
    xn, t = x.detach().double().cpu().numpy(), np.array([[0.0], [1.0], [1.0], [0.0], [1.0]])
    a = xn @ w1.T
    z1 = O.dropout(a, 0.1, l1.seed, 1, b1, True)
    z2 = O.dropout(z1 @ w2.T, 0.1, l2.seed, 1, b2, False)
    s = 1 / (1 + np.exp(-z2))
    np.testing.assert_allclose(y.detach().cpu().numpy(), s, rtol=0, atol=1e-5)
    g2, gb2 = O.dropout_bwd((s - t) / 5, 0.1, l2.seed, 1)
    g1, gb1 = O.dropout_bwd(g2 @ w2, 0.1, l1.seed, 1, z1)
    # 72- and 40-term float32 products, the sigmoid and the loss: some 1e-6 of the largest gradient
    for got, want in ((l2.bias.grad, gb2), (l1.bias.grad, gb1), (l2.weight.grad, g2.T @ z1), (l1.weight.grad, g1.T @ xn), (x.grad, g1 @ w1)):
        got = got.double().cpu().numpy()
        assert np.abs(got - want).max() <= 2e-5 * max(np.abs(want).max(), 1e-3)


@pytest.mark.gpu
def test_two_runs_train_to_the_same_weights_whatever_the_generator(tmp_path):
    class Tiny(nn.Module):
        head_key = "classifier"

        def __init__(self):
            super().__init__()
            self.net = nn.Sequential()
            self.net.add_module("features", nn.Conv2d(3, 2, 3))
            self.net.add_module("classifier", small_head(3))

        backbone = property(lambda self: self.net)

        def forward(self, x):
            return self.net.classifier(F.adaptive_avg_pool2d(self.net.features(x), 6)).squeeze(1)

    g = torch.Generator().manual_seed(0)
    data = [(torch.randn(4, 3, 12, 12, generator=g), torch.randint(0, 2, (4,), generator=g).float()) for _ in range(3)]
    out = []
    for run in range(2):
        torch.manual_seed(11)
        m = Tiny()
        torch.manual_seed(1000 + run)                     # the process's generator differs from run to run
        C.train("driving_constraint", data, None, torch.device("cuda"), str(tmp_path / str(run)), epochs=2, model=m, log=lambda *a: None, dropout_seed=42)
        out.append({k: v.cpu() for k, v in m.state_dict().items()})
    assert all(torch.equal(out[0][k], out[1][k]) for k in out[0])


@pytest.mark.gpu
def test_captured_layers_take_a_step_tensor_and_a_quantised_weight():
    h = small_head(6).cuda()
    heads.counter_dropout(h, 3)
    l1 = h[1].train()
    x = torch.randn(9, 72, generator=torch.Generator().manual_seed(3)).cuda()
    q = nn.Sequential(nn.Linear(72, 8)).cuda()
    heads.mx4_linears(q)
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm), torch.no_grad():
        l1(x)
    torch.cuda.current_stream().wait_stream(warm)
    for layer in (l1, q):                                 # a number as step, a weight not yet quantised: refused, nothing is captured
        graph = torch.cuda.CUDAGraph()
        with torch.no_grad(), pytest.raises(RuntimeError, match="captur"):
            with torch.cuda.graph(graph):
                x.add(1)
                layer(x)
        torch.cuda.synchronize()
    l1.step = torch.zeros((1,), dtype=torch.int64, device="cuda")
    with torch.no_grad():
        q(x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, z = l1(x), q(x)
        for k in (5, 6, 7):
            l1.step.fill_(k)
            graph.replay()
            torch.cuda.synchronize()
            a = F.linear(x, l1.weight).double().cpu().numpy()
            np.testing.assert_allclose(y.cpu().numpy(), O.dropout(a, 0.1, l1.seed, k, l1.bias.double().cpu().numpy(), True), rtol=1e-6, atol=1e-6)
            assert torch.equal(z, q(x))


@pytest.mark.gpu
def test_training_under_autocast():
    h = small_head(7).cuda()
    heads.counter_dropout(h, 4)
    h.train()
    x = torch.randn(5, 72, generator=torch.Generator().manual_seed(4)).cuda()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = h(x)
    y.float().sum().backward()
    assert all(p.grad is not None and p.grad.dtype == torch.float32 and torch.isfinite(p.grad).all() for p in h.parameters())


@pytest.mark.gpu
def test_quantised_head_validates_and_carries_the_image_gradient():
    """eval with four-bit weights against the same layers on the values those bits hold, in float64; the gradient w.r.t. the input straight through"""
    h = small_head(4).eval().cuda()
    ref = [(m.weight.detach().double().cpu().numpy(), m.bias.detach().double().cpu().numpy()) for m in h if isinstance(m, nn.Linear)]
    heads.mx4_linears(h)
    x = torch.randn(6, 72, generator=torch.Generator().manual_seed(2)).cuda().requires_grad_()
    y = h(x)
    (w1, b1), (w2, b2) = [(O.mx4_values(w), b) for w, b in ref]
    z1 = np.maximum(O.mx4_values(x.detach().double().cpu().numpy()) @ w1.T + b1, 0)
    z2 = O.mx4_values(z1.astype(np.float32).astype(np.float64)) @ w2.T + b2
    s = 1 / (1 + np.exp(-z2))
    # an activation within rounding of a 4-bit midpoint may fall to the other side: one step of its block (a quarter of the block's largest at most) times its weight
    np.testing.assert_allclose(y.detach().cpu().numpy(), s, rtol=0, atol=1e-5)
    y.sum().backward()
    want = ((s * (1 - s)) @ w2 * (z1 > 0)) @ w1
    assert np.abs(x.grad.double().cpu().numpy() - want).max() <= 1e-4 * np.abs(want).max()
    assert h[1].weight is None and h[1].codes.shape == (1, 40, 128)               # the float copy is gone
    assert torch.equal(h(x), y)


@pytest.mark.gpu
def test_adopted_detector_head_in_four_bits_under_the_attacks_gradient():
    """a small detector, adopted with linear="mxfp4": the image gradient is the formula's, straight through the quantised head"""
    class Net(nn.Module):
        def __init__(self):
            super().__init__()
            self.conv = nn.Conv2d(3, 8, 3, padding=1)
            self.head = nn.Sequential(nn.Linear(8 * 36, 64), nn.ReLU())
            self.cls = nn.Linear(64, 4)

        def forward(self, x):
            f = F.adaptive_avg_pool2d(torch.relu(self.conv(x)), 6).flatten(1)
            return self.cls(self.head(f))

    torch.manual_seed(5)
    net = Net().eval().cuda()
    x = torch.rand(2, 3, 24, 24, device="cuda")
    report = A.adopt(net, linear="mxfp4", functional=False)
    assert sorted(n for n, w in report["replaced"] if "mxfp4" in w) == ["cls", "head.0"]
    xr = x.clone().requires_grad_()
    logits = net(xr)
    g, = torch.autograd.grad(F.cross_entropy(logits, torch.tensor([1, 2], device="cuda")), xr)
    # the formula, straight through both quantisations, on the values the weights hold
    w1, w2 = net.head[0].held().dequantize().double(), net.cls.held().dequantize().double()
    xf = x.clone().requires_grad_()
    f = F.adaptive_avg_pool2d(torch.relu(net.conv(xf)), 6).flatten(1)
    z = net.head(f).detach()
    # each layer's output on the very values it quantises: a 288- (64-) term float32 sum
    for got, xin, lin, w in ((z, f.detach(), net.head[0], w1), (logits.detach(), z, net.cls, w2)):
        q = torch.tensor(O.mx4_values(xin.double().cpu().numpy())).cuda()
        ref, size = q @ w.t() + lin.bias.double(), q.abs() @ w.t().abs() + lin.bias.double().abs()
        ref = ref.clamp_min(0) if lin.relu else ref
        assert bool(((got.double() - ref).abs() <= (288 / 32 + 16) * 2.0 ** -23 * size + 2.0 ** -24 * ref.abs()).all())
    gl = torch.softmax(logits.detach().double(), 1)
    gl[0, 1] -= 1
    gl[1, 2] -= 1
    gf = ((gl / 2) @ w2 * (z > 0)) @ w1
    want, = torch.autograd.grad(f, xf, gf.float())
    assert float((g - want).abs().max()) <= 1e-4 * float(want.abs().max()) and want.abs().max() > 0
