"""Refusals of the operators around the flow (``nessai_amd.ops``: ``embedding``, ``group_norm_act``, ``grad_norm``,
``clip_grad_norm_``) and of their C entry points.  All of them are decided on the host: no device is needed."""
import ctypes
import math

import pytest
import torch

from nessai_amd import lib, ops


def test_group_norm_act_refuses_what_it_cannot_compute():
    x = torch.randn(4, 5, 12)
    with pytest.raises(ValueError, match="cannot be divided"):
        ops.group_norm_act(x, 5)
    with pytest.raises(ValueError, match="cannot be divided"):
        ops.group_norm_act(x, 0)
    with pytest.raises(ValueError, match="shape"):
        ops.group_norm_act(torch.randn(12), 3)
    with pytest.raises(ValueError, match="Unknown activation"):
        ops.group_norm_act(x, 3, activation="gelu")
    with pytest.raises(ValueError, match="weight"):
        ops.group_norm_act(x, 3, weight=torch.ones(11))
    with pytest.raises(ValueError, match="bias"):
        ops.group_norm_act(x, 3, bias=torch.ones(1, 12))
    with pytest.raises(ValueError, match="eps"):
        ops.group_norm_act(x, 3, eps=-1.0)
    with pytest.raises(ValueError, match="eps"):
        ops.group_norm_act(x, 3, eps=math.nan)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        ops.group_norm_act(x.double(), 3)
    with pytest.raises(TypeError, match="x's type"):
        ops.group_norm_act(x, 3, weight=torch.ones(12, dtype=torch.bfloat16))
    with pytest.raises(TypeError, match="one type"):
        ops.group_norm_act(x.bfloat16(), 3, torch.ones(12), torch.ones(12, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.group_norm_act(x, 3)


def test_embedding_refuses_what_it_cannot_compute():
    w, i = torch.randn(7, 3), torch.tensor([1, 2])
    with pytest.raises(TypeError, match="int32 or int64"):
        ops.embedding(i.float(), w)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        ops.embedding(i, w.double())
    with pytest.raises(ValueError, match="table of shape"):
        ops.embedding(i, w[0])
    with pytest.raises(ValueError, match="table of shape"):
        ops.embedding(i, w[:0])
    for bad in (7, -8):
        with pytest.raises(ValueError, match="padding_idx"):
            ops.embedding(i, w, padding_idx=bad)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.embedding(i, w)


def test_gradient_norm_refuses_what_it_cannot_compute():
    p = torch.nn.Parameter(torch.randn(3))
    assert float(ops.clip_grad_norm_([p], 1.0)) == 0.0 and float(ops.grad_norm([])) == 0.0  # nothing to clip
    p.grad = torch.randn(3)
    with pytest.raises(ValueError, match="norm_type"):
        ops.clip_grad_norm_([p], 1.0, norm_type=3)
    with pytest.raises(ValueError, match="norm_type"):
        ops.grad_norm([p.grad], norm_type=0.5)
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            ops.clip_grad_norm_([p], bad)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.clip_grad_norm_(p, 1.0)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        ops.grad_norm(torch.randn(3, dtype=torch.float64))
    with pytest.raises(TypeError, match="dense"):
        ops.grad_norm(torch.eye(3).to_sparse())


def test_tangents_are_refused():
    """Forward-mode differentiation: the operators have no rule for it, and a result without a tangent reads as a zero."""
    from torch.autograd import forward_ad as fwd

    def dual(t):
        return fwd.make_dual(t, torch.ones_like(t))

    x, w, i = torch.randn(4, 12), torch.ones(12), torch.tensor([1, 2])
    with fwd.dual_level(), torch.no_grad():
        for call in (
            lambda: ops.group_norm_act(dual(x), 3),
            lambda: ops.group_norm_act(x, 3, weight=dual(w)),
            lambda: ops.group_norm_act(x, 3, bias=dual(w)),
            lambda: ops.embedding(i, dual(x)),
            lambda: ops.grad_norm([w, dual(x)]),
        ):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        p = torch.nn.Parameter(torch.zeros(12))
        p.grad = dual(w)
        with pytest.raises(RuntimeError, match="forward-mode"):
            ops.clip_grad_norm_([p], 1.0)
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda v: ops.group_norm_act(v, 3), (x,), (torch.ones_like(x),))
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda v: ops.embedding(i, v), (x,), (torch.ones_like(x),))


def _norm_args(places, sizes, codes):
    n = len(places)
    return (n, (ctypes.c_void_p * n)(*places), (ctypes.c_longlong * n)(*sizes), (ctypes.c_int * n)(*codes))


def test_entry_points_check_their_arguments_before_anything_is_launched():
    L = lib.load()
    ws, out = 4096, 8192  # addresses that no call below reaches
    size = L.nsa_grad_norm_workspace(2, 1000)
    assert L.nsa_grad_norm_workspace(10_000, 10**12) >= size > 0
    for places, sizes, codes, kind, max_norm, bytes_, message in (
        ((16, 32), (4, 5), (0, 7), 2, 1.0, size, b"unknown type"),
        ((16, 32), (4, -1), (0, 0), 2, 1.0, size, b"bad tensor"),
        ((16, None), (4, 1), (0, 0), 2, 1.0, size, b"bad tensor"),
        ((16, 34), (4, 5), (0, 0), 2, 1.0, size, b"aligned"),
        ((16, 32), (4, 5), (0, 0), 9, 1.0, size, b"unknown norm"),
        ((16, 32), (4, 5), (0, 0), 2, -1.0, size, b"max_norm"),
        ((16, 32), (4, 5), (0, 0), 2, math.nan, size, b"max_norm"),
        ((64, 128), (4, 5), (0, 0), 2, 1.0, 7, b"workspace"),
        ((16, 28), (4, 5), (0, 0), 2, 1.0, size, b"overlap"),
        ((16, 16), (4, 4), (0, 0), 2, 1.0, size, b"overlap"),
        ((16, 24), (2, 20), (0, 1), 2, 1.0, 0, b"workspace"),
        ((64, 16), (4, 100), (0, 1), 2, 1.0, size, b"overlap"),
    ):
        args = _norm_args(places, sizes, codes)
        assert L.nsa_grad_clip(*args, kind, max_norm, ws, bytes_, out, None) < 0
        assert message in L.nsa_last_error(), (message, L.nsa_last_error())
    assert L.nsa_group_norm_forward(2, 3, 12, 5, 0, ws, 0, None, None, 1e-5, -1, ws, ws, ws, ws, 1 << 20, None) < 0
    assert b"multiple of groups" in L.nsa_last_error()
    assert L.nsa_group_norm_forward(2, 3, 12, 4, 0, ws, 1, None, None, 1e-5, -1, ws, ws, ws, ws, 1 << 20, None) < 0
    assert L.nsa_group_norm_forward(2, 3, 12, 4, 0, ws, 0, None, None, 1e-5, 7, ws, ws, ws, ws, 1 << 20, None) < 0
    assert L.nsa_group_norm_forward(2, 3, 12, 4, 0, None, 0, None, None, 1e-5, -1, ws, ws, ws, ws, 1 << 20, None) < 0
    assert L.nsa_group_norm_forward(2, 3, 12, 4, 0, ws, 0, None, None, 1e-5, -1, ws, ws, ws, ws, 0, None) < 0
    assert b"workspace" in L.nsa_last_error()
    assert L.nsa_group_norm_backward(2, 3, 12, 4, 0, ws, ws, 0, None, None, -1, ws, ws, ws, None, None, ws, 0, None) < 0
    assert L.nsa_group_norm_workspace(2, 3, 12, 5, 0, 0) == 0
    assert L.nsa_embedding_forward(4, 0, 8, 0, ws, 8, ws, 1.0, ws, None) < 0
    assert L.nsa_embedding_forward(1 << 31, 4, 8, 0, ws, 8, ws, 1.0, ws, None) < 0
    assert L.nsa_embedding_forward(4, 4, 8, 0, ws, 2, ws, 1.0, ws, None) < 0
    assert L.nsa_embedding_backward(4, 4, 8, 0, ws, 8, ws, 1.0, -1, ws, ws, 0, None) < 0
    assert b"workspace" in L.nsa_last_error()
    assert L.nsa_embedding_backward(4, 4, 8, 0, ws, 8, None, 1.0, -1, ws, ws, 1 << 20, None) < 0


def test_group_norm_refuses_channels_that_its_counters_do_not_hold():
    """A group of 2^31 - 1 channels, walked in steps of 256, would pass the last 32-bit number."""
    L, ws = lib.load(), 4096  # (an address that no call below reaches)
    for channels in (2**30 + 1, 2**31 - 1):
        assert L.nsa_group_norm_forward(1, 1, channels, 1, 1, ws, 0, None, None, 1e-5, -1, ws, ws, ws, ws, 1 << 40, None) < 0
        assert b"2^30 channels" in L.nsa_last_error()
        assert L.nsa_group_norm_backward(1, 1, channels, 1, 1, ws, ws, 0, None, None, -1, ws, ws, ws, None, None, ws, 1 << 40, None) < 0
        assert b"2^30 channels" in L.nsa_last_error()
    x = torch.empty(1, dtype=torch.bfloat16).expand(2, 2**30 + 1)
    with pytest.raises(ValueError, match="channels"):
        ops.group_norm_act(x, 1)


def test_group_norm_refuses_more_workgroups_than_a_launch_holds():
    L, ws = lib.load(), 4096
    samples, channels = 2**32, 8209  # (a prime number of groups: a workgroup each, in every sample)
    assert L.nsa_group_norm_forward(samples, 1, channels, channels, 1, ws, 0, None, None, 1e-5, -1, ws, ws, ws, ws, 1 << 62, None) < 0
    assert b"too many samples" in L.nsa_last_error()
    assert L.nsa_group_norm_backward(samples, 1, channels, channels, 1, ws, ws, 0, None, None, -1, ws, ws, ws, None, None, ws, 1 << 62, None) < 0
    assert b"too many samples" in L.nsa_last_error()


def test_operators_of_tensors_without_data():
    """Shapes, types and devices of results on the Meta key, and what a tracer records: the inner operators, whose schemas name
    what they change."""
    from torch.fx.experimental.proxy_tensor import make_fx

    def meta(*shape, dtype=torch.float32, **kw):
        return torch.empty(*shape, dtype=dtype, device="meta", **kw)

    with torch.enable_grad():
        x, w, b = meta(4, 5, 12, dtype=torch.bfloat16, requires_grad=True), meta(12, requires_grad=True), meta(12, requires_grad=True)
        y = ops.group_norm_act(x, 3, w, b, activation="silu")
        assert y.shape == x.shape and y.dtype == torch.bfloat16 and y.is_meta and y.requires_grad
        for wanted in ([x, w, b], [w], [x, b]):
            grads = torch.autograd.grad(y, wanted, torch.empty_like(y), retain_graph=True)
            assert [(g.shape, g.dtype) for g in grads] == [(v.shape, v.dtype) for v in wanted]
        table, ids = meta(7, 3, dtype=torch.float16, requires_grad=True), meta(2, 3, dtype=torch.int32)
        out = ops.embedding(ids, table, scale=2.0, padding_idx=-1)
        assert out.shape == (2, 3, 3) and out.dtype == torch.float16
        (g,) = torch.autograd.grad(out, [table], torch.empty_like(out))
        assert g.shape == table.shape and g.dtype == table.dtype
        p = torch.nn.Parameter(meta(4))
        p.grad = meta(4)
        for norm in (ops.grad_norm([p.grad, meta(3, dtype=torch.bfloat16)]), ops.clip_grad_norm_([p], 1.0)):
            assert norm.shape == () and norm.dtype == torch.float32 and norm.is_meta
        with pytest.raises(ValueError, match="cannot be divided"):
            ops.group_norm_act(x, 5)

        def step(ids, table, w, dy):
            table, w = table.detach().requires_grad_(), w.detach().requires_grad_()
            y = ops.group_norm_act(ops.embedding(ids, table), 4, w)
            grads = torch.autograd.grad(y, [table, w], dy)
            return y, torch.ops.nessai_amd.clip_grad_norm_of_([g.clone() for g in grads], 2, 1.0, False)

        graph = make_fx(step)(meta(5, dtype=torch.int64), meta(7, 8), meta(8), meta(5, 8)).graph
    called = [n.target._schema.name for n in graph.nodes if n.op == "call_function" and "nessai_amd" in str(n.target)]
    assert called == [f"nessai_amd::_{k}" for k in ("embedding_forward", "group_norm_forward", "group_norm_backward",
                                                    "embedding_backward", "clip_gradients_")]
    for name in ("clip_grad_norm_of_", "_clip_gradients_"):
        schema = getattr(torch.ops.nessai_amd, name).default._schema
        assert schema.is_mutable and schema.arguments[0].alias_info.is_write


def test_clip_refuses_a_gradient_with_gaps_given_twice():
    """It is clipped in a copy, of which the entry point's own check knows nothing.  Two views that interleave are apart."""
    wide = torch.empty(6, 40, device="meta")
    p, q = (torch.nn.Parameter(torch.empty(6, 20, device="meta")) for _ in range(2))
    p.grad, q.grad = wide[:, ::2], wide[:, 1::2]
    assert ops.clip_grad_norm_([p, q], 1.0).shape == ()
    with pytest.raises(RuntimeError, match="overlap"):
        ops.clip_grad_norm_([p, p], 1.0)
    q.grad = wide[:, :20]
    with pytest.raises(RuntimeError, match="overlap"):
        ops.clip_grad_norm_([q, p], 1.0)


def test_inner_operators_check_what_their_kernels_rely_on():
    """A traced graph calls them with tensors of its own: strides, shapes, types and devices are checked there as well."""
    def meta(*shape, dtype=torch.float32):
        return torch.empty(*shape, dtype=dtype, device="meta")

    lib.load_torch()
    o = torch.ops.nessai_amd
    x, w, stats = meta(4, 5, 12), meta(12), meta(2, 4, 3)
    wanted = [True, True, True]
    assert o._group_norm_forward(x, w, w, 3, 1e-5, 0)[1].shape == (2, 4, 3)
    assert [g.shape for g in o._group_norm_backward(x, x, w, w, stats, 3, 0, wanted)] == [(4, 5, 12), (12,), (12,)]
    ids, dy = meta(6, dtype=torch.int64), meta(6, 3)
    assert o._embedding_forward(ids, meta(7, 3), 1.0).shape == (6, 3) and o._embedding_backward(dy, ids, 7, 3, 1.0, -1).shape == (7, 3)
    wide = meta(4, 5, 24)[..., ::2]
    for call in (
        lambda: o._group_norm_forward(wide, w, w, 3, 1e-5, 0),
        lambda: o._group_norm_forward(x, meta(24)[::2], None, 3, 1e-5, 0),
        lambda: o._group_norm_forward(x, meta(11), None, 3, 1e-5, 0),
        lambda: o._group_norm_forward(x, w, meta(12, dtype=torch.bfloat16), 3, 1e-5, 0),
        lambda: o._group_norm_forward(x, w, torch.empty(12), 3, 1e-5, 0),
        lambda: o._group_norm_forward(x, w, w, 5, 1e-5, 0),
        lambda: o._group_norm_backward(wide, x, w, w, stats, 3, 0, wanted),
        lambda: o._group_norm_backward(meta(4, 5, 11), x, w, w, stats, 3, 0, wanted),
        lambda: o._group_norm_backward(x.bfloat16(), x, w, w, stats, 3, 0, wanted),
        lambda: o._group_norm_backward(x, x, w, w, meta(4, 3), 3, 0, wanted),
        lambda: o._embedding_forward(ids.int()[::2], meta(7, 3), 1.0),
        lambda: o._embedding_forward(dy, meta(7, 3), 1.0),
        lambda: o._embedding_forward(ids, meta(3, 7).t(), 1.0),
        lambda: o._embedding_backward(meta(3, 6).t(), ids, 7, 3, 1.0, -1),
        lambda: o._embedding_backward(meta(5, 3), ids, 7, 3, 1.0, -1),
        lambda: o._embedding_backward(dy, ids, 0, 3, 1.0, -1),
        lambda: o._total_norm([w, meta(24)[::2]], 2),
        lambda: o._clip_gradients_([w, meta(24)[::2]], 2, 1.0),
    ):
        with pytest.raises(RuntimeError, match="expected"):
            call()
    with pytest.raises(RuntimeError, match="empty list"):  # (the dispatcher's own refusal)
        o._total_norm([], 2)
