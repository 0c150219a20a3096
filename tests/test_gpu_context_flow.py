"""Conditional flows with a trainable net in front of their context (``flows.ContextFlow``): the context's gradient, and the
operators of ``nessai_amd.ops`` together as a training loop uses them, against the oracle's flow and plain torch in float64
(runs on a real MI355X)."""
import math

import numpy as np
import pytest
import torch

from helpers import DEV
from nessai_amd import ops
from nessai_amd.flows import ContextFlow, ContextNet, NeuralSplineFlow, RealNVP
from oracle import flows as O

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _with_grad():
    with torch.enable_grad():  # (the suite's default is no_grad: conftest.py)
        yield


CASES = {
    "nsf_c2": (NeuralSplineFlow, O.NeuralSplineFlow, (6, 16, 2, 2), dict(context_features=2)),
    "rnvp_lu_bn_c1": (RealNVP, O.RealNVP, (5, 24, 3, 1), dict(context_features=1)),
    "nsf_k5_c7_tanh": (NeuralSplineFlow, O.NeuralSplineFlow, (7, 40, 2, 3),
                       dict(context_features=7, num_bins=5, activation=torch.tanh)),
    "nsf_wide_c33": (NeuralSplineFlow, O.NeuralSplineFlow, (8, 68, 3, 2), dict(context_features=33)),
}


def _pair(name, seed=3):
    P, Oc, args, kw = CASES[name]
    torch.manual_seed(seed)
    ref = Oc(*args, **kw)
    with torch.no_grad():
        for n_, p in ref.named_parameters():
            if "linear_layers.1" in n_:
                p.mul_(200.0)
    flow = P(*args, **kw)
    flow.load_state_dict(ref.state_dict())
    flow.to(DEV)
    return ref, flow, args[0], kw["context_features"]


def _plain_net(net, inputs):
    """``ContextNet`` in elementary torch operations (float64, CPU) on copies of its parameters, which are returned too."""
    p = {n: v.detach().cpu().double().requires_grad_(True) for n, v in net.named_parameters()}
    inputs = inputs.cpu().double()
    h = 0.0
    for k, e in enumerate(net.embeddings):
        h = h + p[f"embeddings.{k}.weight"][inputs[:, k].long()] * e.scale
    if net.continuous:
        h = h + inputs[:, len(net.labels) :] @ p["continuous_layer.weight"].t() + p["continuous_layer.bias"]
    for i, norm in enumerate(net.norms):
        h = torch.nn.functional.group_norm(h, norm.num_groups, p[f"norms.{i}.weight"], p[f"norms.{i}.bias"], norm.eps)
        h = {"silu": torch.nn.functional.silu, "tanh": torch.tanh, "relu": torch.relu, None: lambda v: v}[norm.activation](h)
        h = h @ p[f"layers.{i}.weight"].t() + p[f"layers.{i}.bias"]
    return h, p


@pytest.mark.parametrize("training", [False, True], ids=["eval", "train"])
@pytest.mark.parametrize("name", sorted(CASES))
def test_context_gradient_matches_the_oracle(name, training):
    """d loss / d context of both outputs' gradients.  The oracle runs in float32 like the kernels: the two differ by the
    rounding of some hundreds of float32 operations per row, 2e-4 of the largest gradient as in the other gradient tests."""
    ref, flow, D, C = _pair(name)
    ref.train(training)
    flow.train(training)
    x, c = torch.randn(203, D) * 1.3, torch.randn(203, C)
    g_z, g_ld = torch.randn(203, D), torch.randn(203)
    c_ref = c.clone().requires_grad_(True)
    z_ref, ld_ref = ref.forward(x, context=c_ref)
    want = torch.autograd.grad([z_ref, ld_ref], [c_ref, *ref.parameters()], [g_z, g_ld])
    c_dev = c.to(DEV).requires_grad_(True)
    x_dev = x.to(DEV)
    z, ld, _ = flow._run(x_dev, 0, 0, context=c_dev, context_trained=True)
    got = torch.autograd.grad([z, ld], [c_dev, *flow.parameters()], [g_z.to(DEV), g_ld.to(DEV)])
    assert got[0].shape == c.shape and float(want[0].abs().max()) > 1e-3
    for a, b in zip(got, want):
        assert float((a.cpu() - b).abs().max()) <= 2e-4 * max(1e-3, float(b.abs().max()))
    # the other gradients are those of a context without one, bit for bit
    flow2 = type(flow)(*CASES[name][2], **CASES[name][3])
    flow2.load_state_dict(ref.state_dict())
    if not training:
        flow2.to(DEV)
        flow2.eval()
        z, ld, _ = flow2._run(x_dev, 0, 0, context=c.to(DEV))
        plain = torch.autograd.grad([z, ld], list(flow2.parameters()), [g_z.to(DEV), g_ld.to(DEV)])
        assert all(torch.equal(a, b) for a, b in zip(got[1:], plain))


def test_context_gradient_against_differences():
    """Central differences of the float64 oracle along a random direction of the context."""
    ref, flow, D, C = _pair("nsf_c2")
    flow.eval()
    ref = ref.double().eval()
    g = torch.Generator().manual_seed(5)
    x, c, d = (torch.randn(64, k, generator=g) for k in (D, C, C))
    c_dev = c.to(DEV).requires_grad_(True)
    lp = flow._run(x.to(DEV), 0, 1, want_x=False, context=c_dev, context_trained=True)[1]
    (grad,) = torch.autograd.grad(lp.sum(), [c_dev])
    h = 1e-6
    up, down = (float(ref.log_prob(x.double(), context=c.double() + s * h * d.double()).sum().detach()) for s in (1, -1))
    terms = grad.cpu().double() * d.double()
    assert abs((up - down) / (2 * h) - float(terms.sum())) <= 2e-4 * float(terms.abs().sum())


NETS = {
    "labels_and_columns": dict(labels=[4, 7], continuous=3, hidden_features=32, num_groups=4, activation="silu"),
    "labels_alone": dict(labels=[300], hidden_features=20, num_groups=5, num_layers=1, activation="tanh"),
    "columns_alone": dict(continuous=2, hidden_features=24, num_groups=1, num_layers=3, activation="silu"),
}


def _inputs(net, n, seed=0):
    g = torch.Generator().manual_seed(seed)
    cols = [torch.randint(0, k, (n, 1), generator=g).float() for k in net.labels]
    return torch.cat([*cols, torch.randn(n, net.continuous, generator=g)], 1)


@pytest.mark.parametrize("kind", sorted(NETS))
def test_a_training_step_of_flow_and_net_matches_plain_torch(kind):
    """embedding -> group norm + activation -> flow -> loss -> backward -> norm over all tensors -> clip, three steps of
    AdamW: losses, norms and weights against the oracle's flow in float64 under the plain net, clipped by torch."""
    ref, flow, D, C = _pair("nsf_c2")
    ref = ref.double().train()
    torch.manual_seed(1)
    net = ContextNet(C, **NETS[kind])
    both = ContextFlow(flow, net)
    both.to(DEV)
    both.train()
    opt = torch.optim.AdamW(both.parameters(), lr=1e-3)
    _, p = _plain_net(net, _inputs(net, 2))
    opt_ref = torch.optim.AdamW([*ref.parameters(), *p.values()], lr=1e-3)
    for step in range(3):
        x, inputs = torch.randn(500, D, generator=torch.Generator().manual_seed(step)), _inputs(net, 500, seed=step)
        opt.zero_grad()
        loss = -both.log_prob(x.to(DEV), context=inputs.to(DEV)).mean()
        loss.backward()
        grads = {n: q.grad.detach().clone() for n, q in both.named_parameters()}
        norm = ops.clip_grad_norm_(both.parameters(), 0.5)
        opt.step()
        # the reference's parameters: the same leaves, the same expressions
        opt_ref.zero_grad()
        h = _expression(net, p, inputs)
        loss_ref = -ref.log_prob(x.double(), context=h).mean()
        loss_ref.backward()
        wanted = {**{f"flow.{n}": q.grad.clone() for n, q in ref.named_parameters()}, **{f"net.{n}": q.grad.clone() for n, q in p.items()}}
        norm_ref = torch.nn.utils.clip_grad_norm_([*ref.parameters(), *p.values()], 0.5)
        opt_ref.step()
        assert abs(loss.item() - loss_ref.item()) <= 2e-5 * max(1.0, abs(loss_ref.item()))
        assert abs(norm.item() - norm_ref.item()) <= 1e-3 * norm_ref.item()
        if step == 0:  # (later steps: Adam's division by the root of small second moments amplifies roundings)
            for n, g in grads.items():
                w = wanted[n]
                assert float((g.cpu().double() - w).abs().max()) <= 2e-4 * max(1e-3, float(w.abs().max())), n
            assert max(float(g.abs().max()) for n, g in grads.items() if n.startswith("net.")) > 1e-4
    # an element whose gradient is near zero has a step of lr of either sign: at most 3 lr apart, and rarely
    named = dict(both.named_parameters())
    for n, w in {**{f"flow.{k}": v for k, v in ref.named_parameters()}, **{f"net.{k}": v for k, v in p.items()}}.items():
        assert float((named[n].detach().cpu().double() - w.detach()).abs().max()) <= 6.1e-3, n


def _expression(net, p, inputs):
    inputs = inputs.double()
    h = 0.0
    for k, e in enumerate(net.embeddings):
        h = h + p[f"embeddings.{k}.weight"][inputs[:, k].long()] * e.scale
    if net.continuous:
        h = h + inputs[:, len(net.labels) :] @ p["continuous_layer.weight"].t() + p["continuous_layer.bias"]
    for i, norm in enumerate(net.norms):
        h = torch.nn.functional.group_norm(h, norm.num_groups, p[f"norms.{i}.weight"], p[f"norms.{i}.bias"], norm.eps)
        h = {"silu": torch.nn.functional.silu, "tanh": torch.tanh}[norm.activation](h)
        h = h @ p[f"layers.{i}.weight"].t() + p[f"layers.{i}.bias"]
    return h


@pytest.mark.parametrize("kind", sorted(NETS))
def test_three_steps_move_every_weight_as_plain_torch_does(kind):
    """The weights after three clipped steps of AdamW, against float64.  A gradient is off by at most 2e-4 of its tensor's largest
    (the gradient tests); where it is at least 0.02 of that in every step, so by 1 % of itself, the first step is the same to
    rounding (lr times its sign) and the next two, ratios of running means, are off by at most 2 % of lr each: 0.1 lr is
    allowed, where a weight that did not move, or moved the other way, is off by lr at least.  These are a third of the
    weights or more.  Of the others, whose gradients' signs may differ, at most 2 % may be off by more than lr."""
    lr = 1e-3
    ref, flow, D, C = _pair("nsf_c2")
    ref = ref.double().train()
    torch.manual_seed(1)
    net = ContextNet(C, **NETS[kind])
    both = ContextFlow(flow, net)
    both.to(DEV)
    both.train()
    opt = torch.optim.AdamW(both.parameters(), lr=lr)
    _, p = _plain_net(net, _inputs(net, 2))
    named_ref = {**{f"flow.{n}": q for n, q in ref.named_parameters()}, **{f"net.{n}": q for n, q in p.items()}}
    start = {n: q.detach().clone() for n, q in named_ref.items()}
    opt_ref = torch.optim.AdamW(list(named_ref.values()), lr=lr)
    least = {n: torch.full_like(q, math.inf) for n, q in start.items()}
    for step in range(3):
        x, inputs = torch.randn(500, D, generator=torch.Generator().manual_seed(step)), _inputs(net, 500, seed=step)
        opt.zero_grad()
        (-both.log_prob(x.to(DEV), context=inputs.to(DEV)).mean()).backward()
        ops.clip_grad_norm_(both.parameters(), 0.5)
        opt.step()
        opt_ref.zero_grad()
        (-ref.log_prob(x.double(), context=_expression(net, p, inputs)).mean()).backward()
        for n, q in named_ref.items():
            g = q.grad.abs()
            least[n] = torch.minimum(least[n], g / max(1e-3, float(g.max())))
        torch.nn.utils.clip_grad_norm_(list(named_ref.values()), 0.5)
        opt_ref.step()
    named = dict(both.named_parameters())
    assert sorted(named) == sorted(named_ref)
    moved = total = others = far = 0
    for n, q in named_ref.items():
        off = (named[n].detach().cpu().double() - q.detach()).abs()
        sure = least[n] >= 0.02
        assert float(off[sure].max() if sure.any() else 0.0) <= 0.1 * lr, n
        moved, total = moved + int(((q.detach() - start[n]).abs() > 0.5 * lr)[sure].sum()), total + off.numel()
        others, far = others + int((~sure).sum()), far + int((off[~sure] > lr).sum())
    assert moved >= 0.3 * total and far <= 0.02 * others, (moved, total, far, others)


def test_methods_of_a_context_flow_agree():
    torch.manual_seed(2)
    both = ContextFlow(NeuralSplineFlow(4, 16, 2, 2, context_features=3), ContextNet(3, labels=[5], continuous=1))
    both.to(DEV)
    both.eval()
    inputs = _inputs(both.net, 400).to(DEV)
    with torch.inference_mode():
        x, lp = both.sample_and_log_prob(400, context=inputs)
        assert float((both.log_prob(x, context=inputs) - lp).abs().max()) < 5e-4
        z, lp2 = both.forward_and_log_prob(x, context=inputs)
        back, _ = both.inverse(z, context=inputs)
        assert float((back - x).abs().max()) < 1e-4 and both.sample(400, context=inputs).shape == (400, 4)
        z2, ld = both(x, context=inputs)
        assert torch.equal(z, z2) and float((both.base_distribution_log_prob(z) + ld - lp2).abs().max()) < 1e-4
        assert both.log_prob(x[:0], context=inputs[:0]).shape == (0,)
    bad = inputs.clone()
    bad[7, 0] = 5.0  # a label outside the table shows in its row's result, and in no other
    with torch.no_grad():
        lp3 = both.log_prob(x, context=bad)
    assert bool(lp3[7].isnan()) and torch.isfinite(lp3[:7]).all() and torch.isfinite(lp3[8:]).all()
    with pytest.raises(RuntimeError, match="ContextFlow"):  # the flow alone still refuses a context with a gradient
        both.flow.log_prob(x.clone(), context=both.net(inputs.clone()))


def test_labels_that_are_not_whole_numbers_show_in_their_rows():
    """NaN, fractions and infinities are no labels: their rows are NaN, in evaluation and in the net itself, and no other is."""
    torch.manual_seed(2)
    both = ContextFlow(NeuralSplineFlow(4, 16, 2, 2, context_features=3), ContextNet(3, labels=[5], continuous=1))
    both.to(DEV)
    both.eval()
    inputs = _inputs(both.net, 12).to(DEV)
    bad = [math.nan, -0.5, 2.7, 0.9, math.inf, -math.inf, -1.0, 5.0, 2.0**40]
    inputs[: len(bad), 0] = torch.tensor(bad, device=DEV)
    with torch.no_grad():
        assert both.net(inputs)[: len(bad)].isnan().all() and torch.isfinite(both.net(inputs)[len(bad) :]).all()
        lp = both.log_prob(torch.randn(12, 4, device=DEV), context=inputs)
    assert lp[: len(bad)].isnan().all() and torch.isfinite(lp[len(bad) :]).all()


@pytest.mark.parametrize("ftype", ["nsf", "realnvp"])
def test_flow_model_trains_where_one_row_is_left_over(tmp_path, ftype):
    """91 rows in minibatches of 10, which the choice of a batch size accepts; and a training set of one row, refused."""
    from nessai_amd.flowmodel import FlowModel

    rng = np.random.default_rng(3)
    labels = rng.integers(0, 3, size=(91, 1)).astype(float)
    x = rng.normal(size=(91, 2)) + 2.0 * labels
    config = dict(n_inputs=2, n_neurons=8, n_blocks=2, n_layers=1, ftype=ftype,
                  context_net=dict(features=4, labels=[3], hidden_features=16))
    training = dict(max_epochs=3, patience=10, lr=1e-3, batch_size=10, val_size=0.0)
    fm = FlowModel(flow_config=config, training_config=training, output=str(tmp_path), rng=np.random.default_rng(1))
    fm.initialise()
    history = fm.train(x, conditional=labels)
    assert fm._batch_size == 10 and len(history["loss"]) == 3 and np.isfinite(history["loss"]).all()
    before = {k: v.clone() for k, v in fm.model.state_dict().items()}
    with pytest.raises((ValueError, RuntimeError), match="two rows|batch size"):
        fm.train(x[:1], conditional=labels[:1])
    assert all(torch.equal(v, before[k]) for k, v in fm.model.state_dict().items())


@pytest.mark.parametrize("ftype", ["nsf", "realnvp"])
def test_flow_model_trains_a_context_flow_a_context_flow(tmp_path, ftype):
    """``FlowModel.train(conditional=...)`` of a flow with a context net runs, keeps the best weights, saves and reloads."""
    from nessai_amd.flowmodel import FlowModel

    rng = np.random.default_rng(3)
    labels = rng.integers(0, 3, size=(900, 1)).astype(float)
    x = rng.normal(size=(900, 2)) + 2.0 * labels
    config = dict(n_inputs=2, n_neurons=8, n_blocks=2, n_layers=1, ftype=ftype,
                  context_net=dict(features=4, labels=[3], hidden_features=16))
    training = dict(max_epochs=4, patience=10, lr=5e-3, batch_size=200, val_size=0.2, annealing=True)
    fm = FlowModel(flow_config=config, training_config=training, output=str(tmp_path), rng=np.random.default_rng(1))
    fm.initialise()
    with torch.no_grad():  # (as the suite runs: the loop records by itself)
        history = fm.train(x, conditional=labels)
    assert len(history["loss"]) == len(history["val_loss"]) == 4 and np.isfinite(history["loss"]).all()
    assert np.isfinite(history["val_loss"]).all()
    before = fm.log_prob(x[:50], conditional=labels[:50])
    best = -before.mean()
    again = FlowModel(flow_config=config, training_config=training, output=str(tmp_path), rng=np.random.default_rng(1))
    again.load_weights(str(tmp_path / "model.pt"))
    np.testing.assert_allclose(again.log_prob(x[:50], conditional=labels[:50]), before, rtol=0, atol=1e-6)
    assert np.isfinite(best) and fm.sample(20, conditional=labels[:20]).shape == (20, 2)
    z, log_prob = fm.forward_and_log_prob(x[:50], conditional=labels[:50])
    np.testing.assert_allclose(fm.sample_and_log_prob(z=z, conditional=labels[:50])[0], x[:50], atol=1e-3)
    with pytest.raises(ValueError, match="conditional"):
        fm.train(x)
    fm.reset_model(weights=True)
    assert fm._trainer is None
    fm.train(x, conditional=labels, max_epochs=1)
