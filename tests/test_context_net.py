"""``flows.ContextNet`` / ``flows.ContextFlow`` / ``flow_config["context_net"]``: construction and refusals (CPU)."""
import pytest
import torch

from nessai_amd.flows import ContextFlow, ContextNet, Embedding, GroupNormAct, NeuralSplineFlow, RealNVP, configure_model
from nessai_amd.flows.context import label_indices


def test_context_net_checks_its_arguments():
    for kwargs in (dict(features=0, continuous=1), dict(features=2), dict(features=2, labels=[0]),
                   dict(features=2, continuous=-1), dict(features=2, continuous=1, num_layers=0),
                   dict(features=2, continuous=1, hidden_features=30, num_groups=4)):
        with pytest.raises(ValueError):
            ContextNet(**kwargs)
    with pytest.raises(ValueError, match="Unknown activation"):
        ContextNet(2, continuous=1, activation="gelu")
    net = ContextNet(3, labels=[4, 2], continuous=1, hidden_features=16)
    with pytest.raises(ValueError, match="shape"):
        net(torch.zeros(5, 2))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        net(torch.zeros(5, 3))
    table = Embedding(5, 4, padding_idx=2)
    assert not table.weight[2].any() and table.weight[[0, 1, 3, 4]].all()
    assert GroupNormAct(2, 4, activation=torch.nn.functional.silu).activation == "silu"


def test_labels_that_are_not_whole_numbers_have_no_row():
    inf = float("inf")
    values = [0.0, 3.0, -0.5, 0.9, 2.7, 2.0**24 - 1, 2.0**24, 2.0**40, 1e30, inf, -inf, float("nan"), -1.0, -0.0]
    want = [0, 3, -1, -1, -1, 2**24 - 1, -1, -1, -1, -1, -1, -1, -1, 0]
    assert label_indices(torch.tensor(values)).tolist() == want
    assert label_indices(torch.tensor(values, dtype=torch.float64)).tolist()[:8] == want[:6] + [2**24, 2**40]
    for dtype, most in ((torch.float16, 2**11), (torch.bfloat16, 2**8)):
        ids = label_indices(torch.tensor([0.0, 2.5, most - 1, most, inf, float("nan")], dtype=dtype))
        assert ids.dtype == torch.int64 and ids.tolist() == [0, -1, most - 1, -1, -1, -1]
    assert label_indices(torch.tensor([2**30, -3], dtype=torch.int32)).tolist() == [2**30, -3]


def test_inputs_that_cannot_hold_the_labels_are_refused():
    net = ContextNet(2, labels=[3, 2**24 + 1], hidden_features=4, num_groups=1)
    with pytest.raises(ValueError, match="told apart"):
        net(torch.zeros(5, 2))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        net(torch.zeros(5, 2, dtype=torch.int64))
    net = ContextNet(2, labels=[2**8 + 1], hidden_features=4, num_groups=1)
    with pytest.raises(ValueError, match="told apart"):
        net(torch.zeros(5, 1, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        net(torch.zeros(5, 1, dtype=torch.float16))


def test_float64_columns_are_refused():
    """As everywhere in the package; labels alone lose nothing by their type."""
    with pytest.raises(TypeError, match="float64"):
        ContextNet(2, labels=[3], continuous=1, hidden_features=4)(torch.zeros(5, 2, dtype=torch.float64))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ContextNet(2, labels=[3], hidden_features=4)(torch.zeros(5, 1, dtype=torch.float64))


def test_context_flow_from_a_flow_config():
    config = dict(n_inputs=3, n_neurons=8, n_blocks=2, n_layers=1, ftype="nsf",
                  context_net=dict(features=4, labels=[6], continuous=2, hidden_features=8))
    flow = configure_model(config)
    assert isinstance(flow, ContextFlow) and flow.flow.context_features == 4 and isinstance(flow.flow, NeuralSplineFlow)
    names = [n for n, _ in flow.named_parameters()]
    assert any(n.startswith("flow._transform") for n in names) and any(n.startswith("net.embeddings.0") for n in names)
    net = ContextNet(2, continuous=1, hidden_features=8)
    assert configure_model(dict(config, context_net=net)).flow.context_features == 2
    with pytest.raises(TypeError, match="context_net"):
        configure_model(dict(config, context_net="resnet"))
    with pytest.raises(ValueError, match="context features"):
        configure_model(dict(config, context_features=3))
    with pytest.raises(TypeError, match="conditional"):
        ContextFlow(RealNVP(3, 8, 2, 1), net)
    with pytest.raises(ValueError, match="conditional inputs"):
        flow.log_prob(torch.zeros(2, 3))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        flow.log_prob(torch.zeros(2, 3), context=torch.zeros(2, 3))


def test_proposals_refuse_a_context_net(tmp_path):
    from nessai_amd.flowmodel_importance import ImportanceFlowModel
    from nessai_amd.model import RosenbrockModel
    from nessai_amd.proposal import FlowProposal

    config = dict(ftype="nsf", n_inputs=4, context_net=dict(features=2, continuous=1, hidden_features=8))
    proposal = FlowProposal(RosenbrockModel(4), poolsize=10, output=str(tmp_path), flow_config=config)
    with pytest.raises(NotImplementedError, match="context_net"):
        proposal.initialise()
    with pytest.raises(NotImplementedError, match="context_net"):
        ImportanceFlowModel(flow_config=config, output=str(tmp_path)).initialise()


def test_minibatches_of_a_context_flow_have_two_rows_at_least():
    from nessai_amd.train import minibatch_bounds

    assert minibatch_bounds(91, 10) == [*((a, a + 10) for a in range(0, 80, 10)), (80, 91)]
    for n in range(2, 60):
        for size in range(2, 70):
            bounds = minibatch_bounds(n, size)
            assert bounds[0][0] == 0 and bounds[-1][1] == n and all(p[1] == q[0] for p, q in zip(bounds, bounds[1:]))
            assert all(2 <= b - a <= size + 1 for a, b in bounds) and all(b - a == size for a, b in bounds[:-1])
    for n in (0, 1):
        with pytest.raises(ValueError, match="two rows"):
            minibatch_bounds(n, 10)


def test_training_launches_hold_no_memset():
    """They are captured into HIP graphs, where a memset node has given wrong results on later replays: memory is cleared by
    kernels."""
    import os

    import nessai_amd

    csrc = os.path.join(os.path.dirname(nessai_amd.__file__), "csrc")
    names = [n for n in os.listdir(csrc) if n.startswith("nsa_train") and n.endswith((".hip", ".h"))]
    assert len(names) >= 4
    for name in names + ["nsa_embedding.hip", "nsa_group_norm.hip", "nsa_grad_norm.hip"]:
        with open(os.path.join(csrc, name)) as f:
            assert "hipMemset" not in f.read(), name


def test_training_refuses_conditional_inputs_that_are_not_finite(tmp_path):
    import numpy as np

    from nessai_amd.flowmodel import FlowModel

    fm = FlowModel(flow_config=dict(ftype="nsf", n_inputs=2, context_features=1), output=str(tmp_path))
    fm.initialised = True  # (the split is host work: no flow is built for it)
    x, c = np.zeros((20, 2)), np.zeros(20)
    for bad in (np.nan, np.inf):
        c[3] = bad
        for conditional in (c, c[:, None]):
            with pytest.raises(ValueError, match="non-finite conditional"):
                fm.prep_data(x, val_size=0.1, batch_size=5, conditional=conditional)
