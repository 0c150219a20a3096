"""The operators around the flow - ``ops.embedding``, ``ops.group_norm_act``, ``ops.grad_norm``, ``ops.clip_grad_norm_`` -
against plain forms in float64 (runs on a real MI355X).

Tolerances.  u(t) = finfo(t).eps / 2 is the relative error of one rounding to type t.  A result of type t is off by u(t)
of its value from its last rounding, plus what the float32 arithmetic in front of it loses: a sum of float32 terms in a
chain of k additions is off by at most k u(float32) times the sum of the terms' magnitudes.  Where a test uses a factor, the
chain's length is given beside it."""
import math

import pytest
import torch

from helpers import DEV
from nessai_amd import ops

pytestmark = pytest.mark.gpu

U32 = torch.finfo(torch.float32).eps / 2
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(autouse=True)
def _with_grad():
    with torch.enable_grad():  # (the suite's default is no_grad: conftest.py)
        yield


def u(t):
    return torch.finfo(t).eps / 2


def smallest(t):
    """Half the distance of the smallest numbers of the type: what a rounding below the normal range is off by."""
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def randn(*shape, seed=0, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(*shape, generator=g)).to(dtype).to(DEV)


# ---- the norm over many gradients, and the clip -----------------------------------------------------------------------

GRADS = {
    "one_value": [(1,)],
    "one_tensor": [(257, 3)],
    "minibatch_flow": [(16, 64), (64,), (64, 64), (64,), (368, 64), (368,)] * 3,
    "empty_among_them": [(0,), (5,), (0, 4), (7, 1)],
    "many": [(1 + 37 * i % 211,) for i in range(701)],       # several launches
    "tiny": [(1 + 7 * i % 23,) for i in range(577)],
    "large": [(1_000_003,), (3,), (70_001, 5), (1,)],
}


def _params(shapes, dtypes, layout, seed=0):
    """Parameters whose gradients lie side by side in one buffer, apart by odd gaps in it, or in tensors of their own."""
    params, sizes = [], [math.prod(s) for s in shapes]
    total = {t: 0 for t in dtypes}
    places = []
    for i, n in enumerate(sizes):
        t = dtypes[i % len(dtypes)]
        total[t] += 0 if layout == "flat" else 1 + i % 3
        places.append((t, total[t]))
        total[t] += n
    buffers = {t: randn(n + 5, seed=seed, dtype=t, scale=1e-2) for t, n in total.items()}
    for i, (shape, n, (t, at)) in enumerate(zip(shapes, sizes, places)):
        p = torch.nn.Parameter(torch.zeros(shape, dtype=t, device=DEV))
        g = buffers[t][at : at + n].view(shape)
        p.grad = g.clone() if layout == "own" else g
        params.append(p)
    return params, buffers


@pytest.mark.parametrize("layout", ["flat", "gaps", "own"])
@pytest.mark.parametrize("dtypes", [[torch.float32], [torch.bfloat16], [torch.float16], TYPES], ids=["f32", "bf16", "f16", "mixed"])
@pytest.mark.parametrize("norm_type", [2.0, 1.0, math.inf])
@pytest.mark.parametrize("name", sorted(GRADS))
def test_clip_matches_the_definition(name, norm_type, dtypes, layout):
    """Squares and sums are held in 64 bits: the norm is off by its rounding to float32 (and that of the square root:
    2 u).  The factor has three float32 operations, each clipped value one product and one rounding to its type."""
    params, buffers = _params(GRADS[name], dtypes, layout)
    before = [p.grad.double() for p in params]
    kept = {t: b.clone() for t, b in buffers.items()}
    ref = torch.linalg.vector_norm(torch.cat([g.reshape(-1) for g in before]), norm_type)
    alone = ops.grad_norm([p.grad for p in params], norm_type)
    max_norm = 0.3 * float(ref)
    norm = ops.clip_grad_norm_(params, max_norm, norm_type=norm_type)
    assert norm.dtype == torch.float32 and norm.shape == () and norm.device.type == "cuda"
    assert abs(float(norm) - float(ref)) <= 2 * U32 * float(ref) and float(alone) == float(norm)
    factor = max_norm / (float(ref) + 1e-6)
    for p, g in zip(params, before):
        t = p.grad.dtype
        assert bool(((p.grad.double() - g * factor).abs() <= (u(t) + 6 * U32) * (g * factor).abs() + smallest(t)).all())
    if layout == "gaps":  # what lies between the gradients is not theirs
        for t, b in buffers.items():
            inside = torch.zeros(b.numel(), dtype=torch.bool, device=DEV)
            for p in params:
                if p.grad.dtype == t and p.grad.numel():
                    inside[p.grad.storage_offset() : p.grad.storage_offset() + p.grad.numel()] = True
            assert torch.equal(b[~inside], kept[t][~inside])
    # a norm below max_norm leaves every bit as it is
    after = [p.grad.clone() for p in params]
    ops.clip_grad_norm_(params, 1e30, norm_type=norm_type)
    assert all(torch.equal(p.grad, g) for p, g in zip(params, after))


def test_clip_agrees_with_torch_on_values_that_are_not_finite():
    for bad in (math.inf, -math.inf, math.nan):
        for norm_type in (2.0, 1.0, math.inf):
            ours = [torch.nn.Parameter(torch.zeros(5, device=DEV)) for _ in range(3)]
            theirs = [torch.nn.Parameter(torch.zeros(5)) for _ in range(3)]
            for i, (a, b) in enumerate(zip(ours, theirs)):
                b.grad = torch.arange(5.0) - 2.0 + i
                if i == 1:
                    b.grad[3] = bad
                a.grad = b.grad.to(DEV)
            n1 = ops.clip_grad_norm_(ours, 1.0, norm_type=norm_type).cpu()
            n2 = torch.nn.utils.clip_grad_norm_(theirs, 1.0, norm_type=norm_type)
            assert torch.equal(n1, n2) or (n1.isnan() and n2.isnan())
            for a, b in zip(ours, theirs):
                assert torch.allclose(a.grad.cpu(), b.grad, equal_nan=True, rtol=0, atol=0)
            a = torch.nn.Parameter(torch.zeros(2, device=DEV))
            a.grad = torch.tensor([1.0, bad], device=DEV)
            with pytest.raises(RuntimeError, match="non-finite"):
                ops.clip_grad_norm_([a], 1.0, norm_type=norm_type, error_if_nonfinite=True)
            assert float(a.grad[0]) == 1.0  # not touched


def test_norm_of_values_whose_squares_leave_float32():
    for scale in (1e25, 1e-30):
        g = randn(10_000, scale=1.0) * scale
        ref = float(g.double().norm())
        assert abs(float(ops.grad_norm(g)) - ref) <= 2 * U32 * ref


def test_clip_of_gradients_in_other_orders_of_memory():
    base = randn(6, 40, seed=1)
    p = [torch.nn.Parameter(torch.zeros(40, 6, device=DEV)), torch.nn.Parameter(torch.zeros(6, 20, device=DEV)),
         torch.nn.Parameter(torch.zeros(2, 3, 4, 5, device=DEV).contiguous(memory_format=torch.channels_last))]
    wide = randn(6, 40, seed=2)
    p[0].grad, p[1].grad = base.t(), wide[:, ::2]
    p[2].grad = randn(2, 3, 4, 5, seed=3).contiguous(memory_format=torch.channels_last)
    before, others = [q.grad.clone() for q in p], wide[:, 1::2].clone()
    ref = float(torch.cat([g.double().reshape(-1) for g in before]).norm())
    norm = ops.clip_grad_norm_(p, 1.0)
    assert abs(float(norm) - ref) <= 2 * U32 * ref
    for q, g in zip(p, before):
        want = g.double() / (ref + 1e-6)
        assert bool(((q.grad.double() - want).abs() <= 8 * U32 * want.abs()).all())
    assert torch.equal(wide[:, 1::2], others)
    # listed twice: counted twice by the norm, refused by the clip; an expanded gradient cannot be clipped in place
    g = randn(100)
    assert abs(float(ops.grad_norm([g, g])) - math.sqrt(2) * float(g.double().norm())) <= 4 * U32 * 2 * float(g.norm())
    q = torch.nn.Parameter(torch.zeros(100, device=DEV))
    q.grad = g
    with pytest.raises(RuntimeError, match="overlap"):
        ops.clip_grad_norm_([q, q], 1.0)
    q = torch.nn.Parameter(torch.zeros(4, 5, device=DEV))
    q.grad = torch.ones(1, 5, device=DEV).expand(4, 5)
    with pytest.raises(ValueError, match="overlap"):
        ops.clip_grad_norm_([q], 1.0)


def test_clip_of_a_lazy_clone_leaves_its_source():
    for shape in ((100,), (300_001,)):
        source = randn(*shape)
        kept = source.clone()
        p, q = torch.nn.Parameter(torch.zeros(shape, device=DEV)), torch.nn.Parameter(torch.zeros(shape, device=DEV))
        p.grad, q.grad = torch._lazy_clone(source), torch._lazy_clone(source)
        ref = math.sqrt(2) * float(kept.double().norm())
        assert abs(float(ops.clip_grad_norm_([p, q], 0.5)) - ref) <= 4 * U32 * ref
        assert torch.equal(source, kept)
        for g in (p.grad, q.grad):  # (three operations of the factor, one product)
            want = kept.double() * (0.5 / (ref + 1e-6))
            assert bool(((g.double() - want).abs() <= 8 * U32 * want.abs()).all())


def test_clip_is_seen_by_autograd():
    """A graph that saved a gradient notices that the clip changed it."""
    p = torch.nn.Parameter(torch.ones(3, device=DEV))
    p.grad = torch.ones(3, device=DEV)
    v = p.grad._version
    ops.clip_grad_norm_([p], 0.5)
    assert p.grad._version > v


# ---- group norm with an activation ------------------------------------------------------------------------------------

# (shape, groups): rows, short and long sequences, one value per group, one group, widths no vector divides, wide rows
SHAPES = [
    ((1, 8), 2), ((1000, 64), 8), ((333, 20), 5), ((70, 90), 9), ((3, 1, 4), 4), ((2, 7, 6), 6), ((5, 33, 24), 3),
    ((2, 1001, 90), 9), ((4, 16, 16, 32), 8), ((1, 5000, 7), 1), ((3, 2, 3000), 4), ((2, 3, 2100), 1), ((2, 9, 1040), 65),
    ((1, 20_001, 33), 3), ((17, 130, 256), 32), ((4097, 12), 4), ((2, 300, 512), 1), ((3, 40, 2056), 257),
    ((3, 4096), 512), ((2, 4100), 4100), ((2, 3, 1300), 26), ((1040, 150, 64), 4), ((2, 700, 5000), 1),
]
ACTS = [None, "relu", "tanh", "silu"]


def _act64(z, name):
    return {None: lambda v: v, "relu": torch.relu, "tanh": torch.tanh, "silu": lambda v: v * torch.sigmoid(v)}[name](z)


def _group_norm64(x, groups, w, b, eps, act, dy=None):
    """y, and with ``dy`` the gradients, in float64 on the CPU, with what the tolerances need."""
    x64 = x.detach().cpu().double().requires_grad_(True)
    w64 = None if w is None else w.detach().cpu().double().requires_grad_(True)
    b64 = None if b is None else b.detach().cpu().double().requires_grad_(True)
    n, c = x64.shape[0], x64.shape[-1]
    rows = x64.reshape(n, -1, groups, c // groups)
    mean = rows.mean((1, 3), keepdim=True)
    var = ((rows - mean) ** 2).mean((1, 3), keepdim=True)
    z = ((rows - mean) / torch.sqrt(var + eps)).reshape(x64.shape)
    if w64 is not None:
        z = z * w64
    if b64 is not None:
        z = z + b64
    y = _act64(z, act)
    out = dict(y=y.detach(), z=z.detach(), rstd=(1 / torch.sqrt(var + eps)).detach(), mean=mean.detach())
    if dy is not None:
        leaves = [t for t in (x64, w64, b64) if t is not None]
        grads = list(torch.autograd.grad(y, leaves, dy.cpu().double()))
        out["dx"] = grads.pop(0)
        out["dw"] = grads.pop(0) if w64 is not None else None
        out["db"] = grads.pop(0) if b64 is not None else None
    return out


def _close(got, ref, t, lost):
    """Norm-wise: every value is off by its rounding u(t), and the array by ``lost`` of its size from float32 arithmetic."""
    got, ref = got.detach().cpu().double(), ref.detach()
    assert got.shape == ref.shape
    err, size = float((got - ref).norm()), float(ref.norm())
    assert err <= (u(t) + lost) * size + smallest(t) * math.sqrt(max(1, ref.numel())), (err / max(size, 1e-300), u(t), lost)


def _group_norm_case(shape, groups, t, affine, act, seed=0):
    c = shape[-1]
    x = randn(*shape, seed=seed)
    x = (x * torch.exp(0.5 * randn(c, seed=seed + 1)) + 2.0 * randn(c, seed=seed + 2)).to(t)
    w = b = None
    if affine is not None:
        w, b = (1 + 0.3 * randn(c, seed=seed + 3)).to(affine), (0.3 * randn(c, seed=seed + 4)).to(affine)
    return x, w, b, randn(*shape, seed=seed + 5, dtype=t)


@pytest.mark.parametrize("t", TYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("shape,groups", SHAPES, ids=lambda v: "x".join(map(str, v)) if isinstance(v, tuple) else str(v))
def test_group_norm_matches_the_definition(shape, groups, act, t):
    """y, dx, dw, db.  float32 arithmetic: the statistics' chains are at most 128 additions (a thread's values, then its
    wave's), x - mean loses u |x| of a value of size 1 / rstd, and dx is a difference of three terms of at most the size
    of (1 + |xh|) w dy r: all within 128 u (1 + max |x| rstd), norm-wise."""
    for affine in {None, t, torch.float32} if act == "silu" else {torch.float32}:
        x, w, b, dy = _group_norm_case(shape, groups, t, affine, act)
        ref = _group_norm64(x, groups, w, b, 1e-5, act, dy)
        if act == "relu":  # its slope jumps at zero: no upstream gradient where z is within float32 of it
            dy = torch.where(ref["z"].abs() < 1e-3, 0.0, dy.cpu().double()).to(t).to(DEV)
            ref = _group_norm64(x, groups, w, b, 1e-5, act, dy)
        lost = 128 * U32 * (1 + float((x.cpu().double().reshape(shape[0], -1, groups, shape[-1] // groups).abs() * ref["rstd"]).max()))
        leaves = [v.requires_grad_(True) for v in (x, w, b) if v is not None]
        y = ops.group_norm_act(x, groups, w, b, activation=act)
        assert y.dtype == t and y.shape == x.shape and y.is_contiguous()
        _close(y, ref["y"], t, lost)
        grads = list(torch.autograd.grad(y, leaves, dy))
        assert grads[0].dtype == t
        # dx: the three terms may cancel (a group of a few values): relative to the terms, not to their difference
        dx, terms = grads.pop(0).cpu().double(), ref["rstd"].expand(shape[0], 1, groups, shape[-1] // groups)
        wd = (dy.cpu().double().abs() * (1.0 if w is None else w.detach().cpu().double().abs())).reshape(shape[0], -1, groups, shape[-1] // groups)
        size = float((terms * wd).norm())
        err = float((dx - ref["dx"]).norm())
        assert err <= u(t) * float(ref["dx"].norm()) + lost * size + smallest(t) * math.sqrt(dx.numel()), (err, size)
        if w is not None:
            # sums over samples and positions: chains of at most 128 + samples / 4 additions of dz xh and dz
            z = ref["z"]
            count = z.numel() / shape[-1]
            chain = (128 + shape[0] / 4) * U32 + lost
            xh = ((z - b.detach().cpu().double()) / w.detach().cpu().double()).reshape(-1, shape[-1])
            mag = dy.cpu().double().abs().reshape(-1, shape[-1]) * 1.1
            dw, db = (g.cpu().double() for g in grads)
            assert grads[0].dtype == affine and grads[1].dtype == affine
            assert bool(((dw - ref["dw"]).abs() <= u(affine) * ref["dw"].abs() + chain * (mag * (1 + xh.abs())).sum(0) + smallest(affine)).all()), count
            assert bool(((db - ref["db"]).abs() <= u(affine) * ref["db"].abs() + chain * (mag * (1 + xh.abs())).sum(0) + smallest(affine)).all()), count


def test_group_norm_gradients_against_differences():
    """Central differences in float64 of the plain form, of a random direction: truncation h^2, the result's own u."""
    shape, groups = (3, 11, 12), 4
    x, w, b, dy = _group_norm_case(shape, groups, torch.float32, torch.float32, "silu", seed=9)
    leaves = [v.requires_grad_(True) for v in (x, w, b)]
    grads = torch.autograd.grad(ops.group_norm_act(x, groups, w, b, activation="silu"), leaves, dy)
    h = 1e-5
    for k, leaf in enumerate(leaves):
        d = randn(*leaf.shape, seed=20 + k).cpu().double()
        values = []
        for s in (h, -h):
            args = [v.detach().cpu().double() for v in leaves]
            args[k] = args[k] + s * d
            values.append(float((_group_norm64(args[0], groups, args[1], args[2], 1e-5, "silu")["y"] * dy.cpu().double()).sum()))
        slope, ours = (values[0] - values[1]) / (2 * h), float((grads[k].cpu().double() * d).sum())
        assert abs(slope - ours) <= 1e-4 * max(1.0, float((grads[k].cpu().double() * d).abs().sum())), (k, slope, ours)


def test_group_norm_of_values_far_from_zero_and_of_outliers():
    """Statistics about a member of the set: a mean a thousand spreads away, and one value a thousand spreads away,
    cost what rounding x costs (u |x| rstd), not the square of it."""
    for outlier in (False, True):
        x = randn(2, 4001, 16, seed=4)
        if outlier:
            x[:, 0] += 1000.0
        else:
            x = x + 1000.0
        ref = _group_norm64(x, 4, None, None, 1e-5, None)
        y = ops.group_norm_act(x, 4).cpu().double()
        far = float((x.cpu().double().reshape(2, -1, 4, 4).abs() * ref["rstd"]).max())
        assert float((y - ref["y"]).abs().max()) <= 16 * U32 * (1 + far) + 128 * U32 * float(ref["y"].abs().max())


def test_group_norm_of_constant_and_nonfinite_samples():
    x = randn(4, 9, 8, seed=2)
    x[0] = 3.0
    x[1, 4, 0] = math.nan
    x[2, 0, 5] = math.inf
    y = ops.group_norm_act(x, 2, activation="tanh").cpu()
    assert torch.equal(y[0], torch.zeros(9, 8))                   # no spread: zeros, not noise / sqrt(eps)
    assert y[1, :, :4].isnan().all() and torch.isfinite(y[1, :, 4:]).all()
    assert y[2, :, 4:].isnan().all() and torch.isfinite(y[2, :, :4]).all()
    assert torch.isfinite(y[3]).all()


def test_group_norm_takes_views_and_empty_tensors():
    base = randn(6, 10, 48, seed=3)
    for view in (base[:, ::2], base[:, :, 8:40], base.transpose(0, 1), base[1:, 3:], base[:, :, 1:33]):
        ref = _group_norm64(view, 4, None, None, 1e-5, "silu")
        assert float((ops.group_norm_act(view, 4, activation="silu").cpu().double() - ref["y"]).abs().max()) <= 1e-4
    nchw = randn(2, 24, 5, 7, seed=5).contiguous(memory_format=torch.channels_last)
    ours = ops.group_norm_act(nchw.permute(0, 2, 3, 1), 6, activation=None).permute(0, 3, 1, 2)
    theirs = torch.nn.functional.group_norm(nchw.cpu().double(), 6)
    assert float((ours.cpu().double() - theirs).abs().max()) <= 1e-4
    for shape in ((0, 8), (0, 3, 8), (2, 0, 8)):
        x = torch.empty(shape, device=DEV, requires_grad=True)
        w, b = (torch.ones(8, device=DEV, requires_grad=True) for _ in range(2))
        y = ops.group_norm_act(x, 2, w, b, activation="relu")
        grads = torch.autograd.grad(y, [x, w, b], torch.empty(shape, device=DEV))
        assert y.shape == shape and grads[0].shape == shape and not grads[1].any() and not grads[2].any()


def test_group_norm_gradients_of_some_leaves_and_of_an_expanded_upstream():
    x, w, b, _ = _group_norm_case((5, 7, 12), 3, torch.float32, torch.float32, "tanh")
    full = [v.requires_grad_(True) for v in (x, w, b)]
    wanted = torch.autograd.grad(ops.group_norm_act(x, 3, w, b, activation="tanh").sum(), full)
    for k in range(3):
        leaves = [v.detach().requires_grad_(i == k) for i, v in enumerate((x, w, b))]
        (g,) = torch.autograd.grad(ops.group_norm_act(leaves[0], 3, leaves[1], leaves[2], activation="tanh").sum(), [leaves[k]])
        assert torch.equal(g, wanted[k])


def test_group_norm_with_a_weight_or_a_bias_alone():
    x, w, b, dy = _group_norm_case((6, 5, 8), 2, torch.bfloat16, torch.float32, "silu")
    for ww, bb in ((w, None), (None, b)):
        ref = _group_norm64(x, 2, ww, bb, 1e-5, "silu", dy)
        leaf = (ww if ww is not None else bb).requires_grad_(True)
        y = ops.group_norm_act(x, 2, ww, bb, activation="silu")
        (g,) = torch.autograd.grad(y, [leaf], dy)
        _close(y, ref["y"], torch.bfloat16, 1e-5)
        _close(g, ref["dw"] if ww is not None else ref["db"], torch.float32, 1e-5)


# ---- embedding --------------------------------------------------------------------------------------------------------

# (tokens, rows, width, frequencies)
TABLES = [
    (1, 1, 1, "uniform"), (1000, 6, 16, "uniform"), (5000, 1, 8, "uniform"), (777, 300, 5, "uniform"), (64, 70_000, 12, "uniform"),
    (4096, 255, 64, "uniform"), (4097, 256, 33, "uneven"), (9001, 257, 320, "uneven"), (30_000, 65_536, 24, "uneven"),
    (20_000, 40, 100, "one"), (333, 9, 1030, "uniform"), (100_000, 5000, 7, "uneven"), (2048, 100_000, 128, "uniform"),
    (300, 17, 2050, "uneven"), (50_000, 3, 3, "sorted"), (12_345, 700, 48, "sorted"),
    (1_600_003, 3000, 4, "uniform"),
]


def _ids(tokens, rows, how, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    if how == "uneven":
        ids = (torch.exp(torch.rand(tokens, generator=g, dtype=torch.float64) * math.log(rows + 1.0)) - 1).long().clamp(0, rows - 1)
    else:
        ids = torch.randint(0, rows, (tokens,), generator=g)
    if how == "one":
        ids[: tokens - 5] = rows // 2
    if how == "sorted":
        ids = ids.sort().values
    return ids.to(dtype).to(DEV)


@pytest.mark.parametrize("t", TYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("ids_type", [torch.int64, torch.int32], ids=["i64", "i32"])
@pytest.mark.parametrize("tokens,rows,width,how", TABLES)
def test_embedding_matches_the_definition(tokens, rows, width, how, ids_type, t):
    """The lookup is one product and one rounding.  A row of the gradient is a float32 sum: in a chunk of sorted tokens, then
    over the chunks it spans - a chain of at most 64 + tokens / 32 additions, then a product."""
    ids = _ids(tokens, rows, how, ids_type)
    w = randn(rows, width, seed=1, dtype=t).requires_grad_(True)
    dy = randn(tokens, width, seed=2, dtype=t)
    scale, padding = math.sqrt(width), (rows // 2 if how == "uneven" else None)
    out = ops.embedding(ids, w, scale=scale, padding_idx=padding)
    want = w.detach().double()[ids.long()] * scale
    assert out.dtype == t and bool(((out.detach().double() - want).abs() <= (u(t) + 2 * U32) * want.abs() + smallest(t)).all())
    (dw,) = torch.autograd.grad(out, [w], dy)
    assert dw.dtype == t and dw.shape == w.shape
    ref = torch.zeros(rows, width, dtype=torch.float64, device=DEV).index_add_(0, ids.long(), dy.double()) * scale
    mag = torch.zeros(rows, width, dtype=torch.float64, device=DEV).index_add_(0, ids.long(), dy.double().abs()) * scale
    if padding is not None:
        ref[padding] = 0.0
    assert bool(((dw.double() - ref).abs() <= u(t) * ref.abs() + (64 + tokens / 32) * U32 * mag + smallest(t)).all())
    untouched = torch.ones(rows, dtype=torch.bool, device=DEV)
    untouched[ids.long()] = False
    assert not dw[untouched].any() and (padding is None or not dw[padding].any())
    # equal inputs, equal bits
    (again,) = torch.autograd.grad(ops.embedding(ids, w, scale=scale, padding_idx=padding), [w], dy)
    assert torch.equal(dw, again)


# (tokens, rows, width, frequencies): every path of the gradient, runs over many chunks, tables of one to four sorting passes
EXACT_TABLES = [
    (1000, 6, 16, "uniform"), (50_001, 40, 64, "uniform"), (4096, 3000, 24, "uneven"), (4097, 70_001, 12, "uniform"),
    (100_003, 5000, 7, "uneven"), (1_600_003, 3000, 4, "uniform"), (1_600_003, 20_000_000, 2, "uniform"),
    (1_000_003, 5000, 64, "one"), (600_001, 300, 33, "one"), (300_001, 900, 40, "sorted"),
]


@pytest.mark.parametrize("t", TYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("tokens,rows,width,how", EXACT_TABLES)
def test_embedding_gradient_of_whole_numbers_is_exact(tokens, rows, width, how, t):
    """Upstream values of at most 3 in magnitude and at most a million tokens in a row: every sum is a whole number below
    2^24, exact in float32 in any order, so that one token lost, doubled or misplaced shows.  One rounding to the type."""
    ids = _ids(tokens, rows, how, torch.int64)
    dy = torch.randint(-3, 4, (tokens, width), generator=torch.Generator().manual_seed(7)).to(DEV)
    dy[:, 0] = 1 + torch.arange(tokens, device=DEV) % 3  # (a column that cannot cancel)
    w = torch.zeros(rows, width, dtype=t, device=DEV, requires_grad=True)
    padding = rows // 3 if how == "uneven" else None
    (dw,) = torch.autograd.grad(ops.embedding(ids, w, scale=0.25, padding_idx=padding), [w], dy.to(t))
    want = torch.zeros(rows, width, dtype=torch.int64, device=DEV).index_add_(0, ids, dy)
    if padding is not None:
        want[padding] = 0
    assert int(want.abs().max()) < 2**24
    assert torch.equal(dw, (want.float() * 0.25).to(t))


def test_embedding_of_a_transposed_table():
    w = randn(11, 8, seed=1)
    ids = torch.randint(0, 8, (3, 4, 5), generator=torch.Generator().manual_seed(2)).to(DEV)
    leaf = w.clone().requires_grad_(True)
    out = ops.embedding(ids, leaf.t())  # 8 rows of 11
    assert torch.equal(out.detach(), w.t()[ids])
    dy = torch.randint(-3, 4, (3, 4, 5, 11), generator=torch.Generator().manual_seed(3)).float().to(DEV)
    (dw,) = torch.autograd.grad(out, [leaf], dy)
    assert torch.equal(dw, torch.zeros(8, 11, device=DEV).index_add_(0, ids.reshape(-1), dy.reshape(-1, 11)).t())


def test_embedding_of_indices_outside_the_table():
    """Such a row is NaN, takes no part in the gradient, and leaves every other row as it is."""
    w = randn(10, 6, seed=1).requires_grad_(True)
    ids = torch.tensor([3, 10, -1, 0, 2**40, -(2**40), 9], device=DEV)
    out = ops.embedding(ids, w, scale=2.0)
    bad = (ids < 0) | (ids >= 10)
    assert out[bad].isnan().all() and torch.equal(out[~bad], w.detach()[ids[~bad]] * 2.0)
    (dw,) = torch.autograd.grad(out, [w], torch.ones_like(out))
    want = torch.zeros(10, 6, device=DEV)
    want[[0, 3, 9]] = 2.0
    assert torch.equal(dw, want)
    out = ops.embedding(torch.tensor([2**31 - 1, -(2**31)], dtype=torch.int32, device=DEV), w)
    assert out.isnan().all()
    (dw,) = torch.autograd.grad(out, [w], torch.ones_like(out))
    assert not dw.any()


def test_second_derivatives_are_refused():
    x, w, b, dy = _group_norm_case((3, 4, 8), 2, torch.float32, torch.float32, "silu")
    y = ops.group_norm_act(x.requires_grad_(True), 2, w, b, activation="silu")
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(y, [x], dy, create_graph=True)
    table = randn(5, 4).requires_grad_(True)
    out = ops.embedding(torch.tensor([1, 2], device=DEV), table)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(out, [table], torch.ones_like(out), create_graph=True)


def test_embedding_shapes_views_and_padding():
    w = randn(11, 8, seed=1)
    ids = torch.randint(0, 11, (3, 4, 5), device=DEV)
    assert torch.equal(ops.embedding(ids, w), w[ids])
    assert torch.equal(ops.embedding(ids.transpose(0, 2), w), w[ids.transpose(0, 2)])
    assert torch.equal(ops.embedding(ids[0, 0, 0], w), w[ids[0, 0, 0]])
    assert torch.equal(ops.embedding(ids, w[:, 1:6]), w[:, 1:6][ids])
    assert torch.equal(ops.embedding(ids, w.t()[:, :8].t()), w[:8][ids]) if int(ids.max()) < 8 else True
    assert ops.embedding(ids[:0], w).shape == (0, 4, 5, 8)
    leaf = w.clone().requires_grad_(True)
    out = ops.embedding(ids[:0], leaf)
    (dw,) = torch.autograd.grad(out, [leaf], torch.empty_like(out))
    assert dw.shape == leaf.shape and not dw.any()
    # a table that is a view gets its gradient through the view; an expanded upstream gradient
    leaf = w.clone().requires_grad_(True)
    (dw,) = torch.autograd.grad(ops.embedding(ids, leaf[:, 2:5], padding_idx=-1).sum(), [leaf])
    counts = torch.bincount(ids.reshape(-1), minlength=11).float()
    counts[10] = 0.0
    assert torch.equal(dw[:, 2:5], counts[:, None].expand(11, 3)) and not dw[:, :2].any() and not dw[:, 5:].any()


# ---- streams, graphs --------------------------------------------------------------------------------------------------


def _chain(ids, table, w, b, dy):
    """A pass through all operators, as a training step makes it; returns everything it computes."""
    h = ops.embedding(ids, table, scale=2.0)
    y = ops.group_norm_act(h, 4, w, b, activation="silu")
    grads = torch.autograd.grad(y, [table, w, b], dy)
    params = []
    for leaf, g in zip((table, w, b), grads):
        p = torch.nn.Parameter(leaf.detach())
        p.grad = g
        params.append(p)
    norm = ops.clip_grad_norm_(params, 0.5)
    return [y.detach(), norm, *[p.grad for p in params]]


def _chain_inputs(seed, tokens=3000, rows=50, width=32):
    ids = torch.randint(0, rows, (tokens,), generator=torch.Generator().manual_seed(seed)).to(DEV)
    leaves = [randn(rows, width, seed=seed), 1 + 0.1 * randn(width, seed=seed + 1), 0.1 * randn(width, seed=seed + 2)]
    return [ids, *[v.requires_grad_(True) for v in leaves], randn(tokens, width, seed=seed + 3)]


def test_two_streams_at_once():
    want = [[t.clone() for t in _chain(*_chain_inputs(s))] for s in (1, 2)]
    inputs = [_chain_inputs(s) for s in (1, 2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(5):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k] = _chain(*inputs[k])
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_two_captured_graphs_replayed_between_eager_calls():
    inputs = [_chain_inputs(s) for s in (3, 4)]
    want = [[t.clone() for t in _chain(*i)] for i in inputs]
    torch.cuda.synchronize()
    graphs, outs = [], []
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):  # warm up off the default stream, as torch asks
        for i in inputs:
            _chain(*i)
    torch.cuda.synchronize()
    for i in inputs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_chain(*i))
        graphs.append(g)
    for _ in range(3):
        for g in graphs:
            g.replay()
        eager = _chain(*inputs[0])
        torch.cuda.synchronize()
        for a, b in zip(want, outs):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
        assert all(torch.equal(x, y) for x, y in zip(want[0], eager))
    # a replay reads new values from the same places
    with torch.no_grad():
        inputs[0][4].mul_(0.5)
    fresh = [t.clone() for t in _chain(*inputs[0])]
    graphs[0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(fresh, outs[0]))


def test_a_leaf_changed_before_its_backward_pass_is_noticed():
    x, w, b, dy = _group_norm_case((6, 5, 8), 2, torch.float32, torch.float32, "silu")
    w.requires_grad_(True)
    y = ops.group_norm_act(x, 2, w, b, activation="silu")
    with torch.no_grad():
        w.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, [w], dy)


@pytest.mark.parametrize("t", TYPES, ids=["f32", "bf16", "f16"])
def test_unaligned_tensors(t):
    """Every tensor begins one element behind a 16-byte border: the accesses narrow, the results stay."""
    def behind(v):
        room = torch.empty(v.numel() + 1, dtype=v.dtype, device=DEV)
        room[1:].copy_(v.reshape(-1))
        return room[1:].view(v.shape)

    for shape, groups in (((300, 64), 8), ((3, 700, 64), 16), ((2, 3, 40), 5)):
        x, w, b, dy = _group_norm_case(shape, groups, t, t, "silu")
        results = []
        for f in (lambda v: v, behind):
            leaves = [f(v.detach()).requires_grad_(True) for v in (x, w, b)]
            y = ops.group_norm_act(leaves[0], groups, leaves[1], leaves[2], activation="silu")
            results.append([y, *torch.autograd.grad(y, leaves, f(dy))])
        for p, q in zip(*results):
            # the same arithmetic in another order: float32 sums of at most 128 + samples additions, then a rounding
            assert float((p.double() - q.double()).norm()) <= (2 * u(t) + 1e-5) * float(p.double().norm())
    for rows, width in ((9, 64), (900, 64), (900, 40)):
        ids = _ids(2000, rows, "uneven", torch.int64)
        w, dy = randn(rows, width, dtype=t), randn(2000, width, seed=1, dtype=t)
        results = []
        for f in (lambda v: v, behind):
            leaf = f(w).requires_grad_(True)
            out = ops.embedding(ids, leaf, scale=3.0)
            results.append([out, *torch.autograd.grad(out, [leaf], f(dy))])
        assert torch.equal(results[0][0], results[1][0])
        assert float((results[0][1].double() - results[1][1].double()).norm()) <= (2 * u(t) + 1e-5) * float(results[0][1].double().norm())


# ---- offsets beyond 32 bits -------------------------------------------------------------------------------------------


def test_norm_and_clip_of_a_tensor_of_more_than_two_to_the_31_elements():
    n = 2**31 + 1001  # (4.3 GB; longer than one launch's share of elements)
    p = torch.nn.Parameter(torch.empty(n, dtype=torch.bfloat16, device=DEV))
    p.grad = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    places = [0, 5, 2**31 - 1, 2**31, n - 1]
    p.grad[places] = 2.0
    assert abs(float(ops.grad_norm(p.grad)) - math.sqrt(20.0)) <= 2 * U32 * math.sqrt(20.0)
    ops.clip_grad_norm_([p], 1.0)
    want = torch.tensor(2.0 / (math.sqrt(20.0) + 1e-6)).bfloat16()
    assert bool((p.grad[places].cpu() == want).all()) and int(torch.count_nonzero(p.grad)) == len(places)


def test_embedding_in_a_table_of_more_than_two_to_the_31_elements():
    rows, width = 2_200_000, 1024  # (4.5 GB)
    w = torch.zeros(rows, width, dtype=torch.bfloat16, device=DEV)
    ids = torch.tensor([rows - 1, 0, 2_097_152, rows - 1, 7] * 30, device=DEV)
    w[ids.unique()] = randn(4, width).bfloat16()
    w.requires_grad_(True)
    out = ops.embedding(ids, w)
    assert torch.equal(out.detach(), w.detach()[ids])
    dy = randn(len(ids), width, seed=1, dtype=torch.bfloat16)
    (dw,) = torch.autograd.grad(out, [w], dy)
    for row in (rows - 1, 0, 2_097_152, 7):
        ref = dy.double()[ids == row].sum(0)
        mag = dy.double()[ids == row].abs().sum(0)
        assert bool(((dw[row].double() - ref).abs() <= u(torch.bfloat16) * ref.abs() + 100 * U32 * mag).all())  # (60 terms)
    assert int(torch.count_nonzero(dw.abs().amax(1))) == 4


@pytest.mark.parametrize("shape", [(3, 1_500_001, 512), (36_000_000, 64)], ids=["long", "rows"])
def test_group_norm_of_more_than_two_to_the_31_elements(shape):
    """The last sample (or rows) agrees with itself alone: other chunks, the same sums to 128 u per chain, then a rounding."""
    x = torch.empty(shape, dtype=torch.bfloat16, device=DEV).normal_(generator=torch.Generator(device=DEV).manual_seed(1))
    y = ops.group_norm_act(x, 8, activation="silu")
    tail = slice(-1, None) if len(shape) == 3 else slice(-1000, None)
    alone = ops.group_norm_act(x[tail].clone(), 8, activation="silu")
    assert float((y[tail].double() - alone.double()).norm()) <= (2 * u(torch.bfloat16) + 128 * U32) * float(alone.double().norm())
    leaf = x.requires_grad_(True)
    (dx,) = torch.autograd.grad(ops.group_norm_act(leaf, 8, activation="silu"), [leaf], y)
    end = x.detach()[tail].clone().requires_grad_(True)
    (want,) = torch.autograd.grad(ops.group_norm_act(end, 8, activation="silu"), [end], y[tail].clone())
    assert float((dx[tail].double() - want.double()).norm()) <= (2 * u(torch.bfloat16) + 1e-4) * float(want.double().norm())


# ---- launches of more workgroups than one dimension holds -------------------------------------------------------------


def test_group_norm_of_more_than_two_to_the_24_groups_of_samples():
    """8193 x 2048 (sample, group) pairs.  The first and last samples agree with themselves alone bit for bit: the same chunks.
    bias: a float32 sum of 3 terms per sample, then 64 bits and a rounding.  weight: xh = (x - mean) rstd of three values; the
    mean is off by 3 u max|x|, the root by twice that, so xh, of at most sqrt(3), by 16 u (1 + max|x| rstd)."""
    shape, groups = (8193, 3, 2048), 2048
    x, w, b, dy = _group_norm_case(shape, groups, torch.bfloat16, torch.float32, None)
    leaves = [v.requires_grad_(True) for v in (x, w, b)]
    y = ops.group_norm_act(x, groups, w, b)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    for part in (slice(0, 2), slice(-2, None)):
        xs = x.detach()[part].clone().requires_grad_(True)
        ys = ops.group_norm_act(xs, groups, w, b)
        assert torch.equal(ys, y[part])
        assert torch.equal(torch.autograd.grad(ys, [xs], dy[part].clone())[0], dx[part])
    assert torch.isfinite(dx).all()
    d, v = dy.double(), x.detach().double()
    rstd = 1 / torch.sqrt(v.var(1, correction=0, keepdim=True) + 1e-5)
    xh = (v - v.mean(1, keepdim=True)) * rstd
    assert bool(((db.double() - d.sum((0, 1))).abs() <= 4 * U32 * d.abs().sum((0, 1))).all())
    tol = (d.abs() * 16 * U32 * (1 + v.abs().amax(1, keepdim=True) * rstd)).sum((0, 1))
    assert bool(((dw.double() - (d * xh).sum((0, 1))).abs() <= tol + U32 * dw.abs()).all())


def test_group_norm_of_more_than_two_to_the_24_slabs():
    """A prime number of groups of one channel: 2056 x 8209 workgroups of one channel each, in every pass."""
    shape, groups = (2056, 2, 8209), 8209
    x, w, b, dy = _group_norm_case(shape, groups, torch.bfloat16, torch.float32, None)
    leaves = [v.requires_grad_(True) for v in (x, w, b)]
    y = ops.group_norm_act(x, groups, w, b, activation="silu")
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    for part in (slice(0, 1), slice(-1, None)):
        xs = x.detach()[part].clone().requires_grad_(True)
        ys = ops.group_norm_act(xs, groups, w, b, activation="silu")
        assert torch.equal(ys, y[part])
        assert torch.equal(torch.autograd.grad(ys, [xs], dy[part].clone())[0], dx[part])
    # of two values, xh is their difference over its own size: 1 / sqrt(1 + eps / var), by the formula of the tests above
    v, d = x.detach().double(), dy.double()
    rstd = 1 / torch.sqrt(v.var(1, correction=0, keepdim=True) + 1e-5)
    xh = (v - v.mean(1, keepdim=True)) * rstd
    z = xh * w.detach().double() + b.detach().double()
    s = torch.sigmoid(z)
    dz, lost = d * s * (1 + z * (1 - s)), 16 * U32 * (1 + v.abs().amax(1, keepdim=True) * rstd)
    # silu and its slope change by at most 1.1 and 0.5 times what z is off by; their own arithmetic loses less than 16 u (1 + |z|)
    far = w.detach().double().abs() * lost + 16 * U32 * (1 + z.abs())
    assert bool(((y.double() - z * s).abs() <= u(torch.bfloat16) * (z * s).abs() + 1.2 * far + smallest(torch.bfloat16)).all())
    size = (d.abs() * (far + lost)).sum((0, 1))
    assert bool(((db.double() - dz.sum((0, 1))).abs() <= size).all()) and bool(((dw.double() - (dz * xh).sum((0, 1))).abs() <= 2 * size).all())


def test_group_norm_launches_in_two_dimensions():
    """More than 2^20 workgroups of rows (one element a lane: an odd address) and of samples in tiles, and of channels."""
    rows = 2**24 + 4097
    room = torch.empty(rows * 64 + 1, dtype=torch.bfloat16, device=DEV).normal_(generator=torch.Generator(device=DEV).manual_seed(3))
    x = room[1:].view(rows, 64)
    y = ops.group_norm_act(x, 8, activation="silu")
    for part in (slice(0, 1000), slice(-5000, None)):
        alone = ops.group_norm_act(x[part].clone(), 8, activation="silu")
        # (16-byte accesses there: another order of 8 additions)
        assert float((y[part].double() - alone.double()).norm()) <= (2 * u(torch.bfloat16) + 128 * U32) * float(alone.double().norm())
    del room, x, y
    samples = 2**20 + 5
    x = torch.empty(samples, 4100, dtype=torch.bfloat16, device=DEV).normal_(generator=torch.Generator(device=DEV).manual_seed(4))
    y = ops.group_norm_act(x, 41, activation="tanh")
    for part in (slice(0, 3), slice(2**20 - 1, None)):
        assert torch.equal(ops.group_norm_act(x[part].clone(), 41, activation="tanh"), y[part])
    del x, y
    c = 2**24 + 1024
    x, dy = randn(2, c, seed=5), randn(2, c, seed=6)
    w, b = torch.ones(c, device=DEV, requires_grad=True), torch.zeros(c, device=DEV, requires_grad=True)
    dw, db = torch.autograd.grad(ops.group_norm_act(x, 64, w, b), [w, b], dy)
    v, d = x.double().view(2, 64, -1), dy.double()
    xh = ((v - v.mean(2, keepdim=True)) / torch.sqrt(v.var(2, correction=0, keepdim=True) + 1e-5)).view(2, c)
    # (two terms; a chain of 257 values in a thread's sums, about a member of at most 6 spreads)
    assert bool(((db.double() - d.sum(0)).abs() <= 2 * U32 * d.abs().sum(0)).all())
    assert bool(((dw.double() - (d * xh).sum(0)).abs() <= 260 * U32 * (1 + 6) * (d.abs() * (1 + xh.abs())).sum(0)).all())


# ---- traced ------------------------------------------------------------------------------------------------------------


def test_a_compiled_pass_gives_the_eager_bits():
    """torch.compile without a code generator: the traced graphs of the forward and the backward pass, run as they are."""
    def forward(ids, table, w, b):
        return ops.group_norm_act(ops.embedding(ids, table, scale=2.0), 4, w, b, activation="silu")

    ids, table, w, b, dy = _chain_inputs(5)
    want = [y := forward(ids, table, w, b), *torch.autograd.grad(y, [table, w, b], dy)]
    compiled = torch.compile(forward, backend="aot_eager", fullgraph=True)
    got = [y := compiled(ids, table, w, b), *torch.autograd.grad(y, [table, w, b], dy)]
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    with torch.no_grad():
        assert torch.equal(compiled(ids, table, w, b), want[0])


def test_a_compiled_clip_of_parameters():
    """The gradients of parameters that a compiled function is given."""
    params, _ = _params(GRADS["minibatch_flow"], [torch.float32], "own")
    others, _ = _params(GRADS["minibatch_flow"], [torch.float32], "own")
    want = ops.clip_grad_norm_(params, 0.5)
    got = torch.compile(lambda ps: ops.clip_grad_norm_(ps, 0.5), backend="aot_eager")(others)
    assert torch.equal(want, got) and all(torch.equal(p.grad, q.grad) for p, q in zip(params, others))


def test_a_compiled_clip_changes_the_gradients():
    def clip(grads):
        return torch.ops.nessai_amd.clip_grad_norm_of_(grads, 2, 0.5, False)

    for dtypes in ([torch.float32], TYPES):
        params, _ = _params(GRADS["minibatch_flow"], dtypes, "own")
        ours = [p.grad.clone() for p in params]
        want = ops.clip_grad_norm_(params, 0.5)
        got = torch.compile(clip, backend="aot_eager", fullgraph=True)(ours)
        assert torch.equal(want, got) and all(torch.equal(p.grad, g) for p, g in zip(params, ours))
