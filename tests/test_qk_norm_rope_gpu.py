"""Norms of query and key heads with their rotation in one pass, forward and
backward, against the formulas in float64: widths of one pair, odd numbers of
pairs and every lane count, q and k apart and as columns of one product,
positions far out, and rows that are not whole 16-byte chunks."""
from math import pi

import numpy as np
import pytest

from qutai_amd import Tensor
from qutai_amd.backends import amd, amd_lm
from qutai_amd.lm import Config, Decoder, autocast, qk_norm_rope
from tests.helpers import download, stored, upload

pytestmark = pytest.mark.gpu

THETA, EPS = 10000.0, 1e-6
UNIT = 2.0 ** -24  # half a step of fp32
STEP = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8}

CASES = [
    # dtype, batch, time, heads, kv_heads, dim, stacked, starts, offset
    ("float32", 1, 1, 1, 1, 2, False, None, 0),
    ("float32", 2, 3, 4, 2, 6, True, None, 5),
    ("float32", 1, 5, 3, 1, 64, False, [123456], 0),
    ("float32", 2, 17, 5, 5, 80, True, None, 0),
    ("float32", 3, 9, 2, 1, 128, False, [0, 7, 100000], 1),
    ("float32", 1, 4, 2, 2, 254, False, None, 0),
    ("float32", 1, 3, 2, 2, 256, True, None, 900000),
    ("bfloat16", 1, 1, 1, 0, 2, False, None, 0),
    ("bfloat16", 2, 3, 4, 2, 6, True, [3, 4], 0),
    ("bfloat16", 8, 1, 16, 4, 64, True, [1000, 1, 0, 999, 31, 32, 33, 500], 0),
    ("bfloat16", 2, 67, 16, 4, 64, True, None, 0),
    ("bfloat16", 3, 33, 6, 3, 80, False, None, 2),
    ("bfloat16", 1, 70, 9, 3, 96, True, None, 0),
    ("bfloat16", 2, 40, 8, 8, 128, False, [5, 60000], 0),
    ("bfloat16", 1, 3, 0, 2, 256, False, None, 0),
    ("bfloat16", 5, 600, 3, 1, 32, True, None, 0),
    ("bfloat16", 1, 7, 3, 2, 8, True, None, 0),
]


def turned(values, angle, sign):
    even, odd = values[..., 0::2], values[..., 1::2]
    out = np.empty_like(values)
    out[..., 0::2] = even * np.cos(angle) - sign * odd * np.sin(angle)
    out[..., 1::2] = sign * even * np.sin(angle) + odd * np.cos(angle)
    return out


def pair_sums(values):
    return np.repeat(np.abs(values[..., 0::2]) + np.abs(values[..., 1::2]), 2, axis=-1)


def reference(x, w, angle, g=None):
    """((y, its bound), and with g ((dx, bound), (dw, sum of magnitudes)))."""
    dim = x.shape[-1]
    if w is None:
        r, unit, w = np.ones(x.shape[:-1] + (1,)), x, np.ones(dim)
        normed = False
    else:
        r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + EPS)
        unit, normed = x * r, True
    n = unit * w
    y = turned(n, angle, 1)
    # r: dim squares, their sum, mean, eps, root and quotient; two products; a turn of two products whose
    # sine and cosine are off by the angle's rounding (half a turn at most) and two units of their own
    wide = (dim / 2 + 4) * UNIT
    turn = (pi + 4 + 2) * UNIT
    y_bound = pair_sums(n) * (wide + 3 * UNIT + turn)
    if g is None:
        return y, y_bound
    gn = turned(g, angle, -1)
    gn_bound = pair_sums(g) * turn
    t, t_bound = gn * w, (gn_bound + UNIT * np.abs(gn)) * np.abs(w)
    if not normed:
        return (y, y_bound), (gn, gn_bound), None
    mean = (t * unit).mean(-1, keepdims=True)
    size = (np.abs(t) * np.abs(unit)).mean(-1, keepdims=True)
    mean_bound = (t_bound * np.abs(unit)).mean(-1, keepdims=True) + size * (2 * wide + dim * UNIT)
    dx = r * (t - unit * mean)
    dx_bound = r * (t_bound + np.abs(unit) * (mean_bound + size * (wide + 3 * UNIT)) + np.abs(t) * (wide + 3 * UNIT))
    axes = tuple(range(x.ndim - 1))
    dw, terms = (gn * unit).sum(axes), (np.abs(gn) * np.abs(unit)).sum(axes)
    dw_bound = (gn_bound * np.abs(unit)).sum(axes) + terms * (wide + 2 * UNIT)
    return (y, y_bound), (dx, dx_bound), (dw, dw_bound, terms)


def within(got, expected, bound, dtype):
    step = STEP[dtype]
    limit = bound + step * (np.abs(expected) + bound)
    worst = np.max(np.abs(got - expected) - limit)
    assert (np.abs(got - expected) <= limit).all(), worst


@pytest.mark.parametrize("normed", [True, False])
@pytest.mark.parametrize("dtype,batch,time,heads,kv_heads,dim,stacked,starts,offset", CASES)
def test_forward_and_backward_match_float64(dtype, batch, time, heads, kv_heads, dim, stacked, starts, offset, normed):
    rng = np.random.default_rng(dim + time)
    positions, wide = batch * time, (heads * dim, kv_heads * dim)
    total = wide[0] + 2 * wide[1] + 3  # odd pitch for the odd widths
    total += -total % 8 if dim % 8 == 0 else 0
    at = offset + np.arange(time)[None] + np.array([0] * batch if starts is None else starts)[:, None]
    angle = at.reshape(-1, 1, 1) * THETA ** (-np.arange(0, dim, 2) / dim)
    place = dict(offset=offset)
    if starts is not None:
        place["starts"] = amd.storage(starts, dtype="int64")
    if stacked:
        block = rng.standard_normal((positions, total)) * 2
        source = upload(block, dtype)
        block = stored(block, dtype)
        rows = [block[:, :wide[0]], block[:, wide[0]:wide[0] + wide[1]]]
        inputs = (source, source)
        place.update(q_row=total, k_column=wide[0], k_row=total)
    else:
        rows = [rng.standard_normal((positions, n)) * 2 for n in wide]
        inputs = tuple(upload(x, dtype) if x.size else None for x in rows)
        rows = [stored(x, dtype) for x in rows]
    weights = [(1 + 0.1 * rng.standard_normal(dim)).astype(np.float32) if normed else None for _ in range(2)]
    held = [None if w is None else upload(w, "float32") for w in weights]
    dims = (batch, time, heads, kv_heads, dim, THETA, EPS)
    out = amd_lm.qk_norm_rope(*inputs, *held, *dims, **place)
    gradients = [stored(rng.standard_normal((positions, n)), dtype) for n in wide]
    given = [upload(g, dtype) if g.size else None for g in gradients]
    target = upload(np.full((positions, total), 7.0), dtype) if stacked else None
    back = amd_lm.qk_norm_rope_backward(*given, *inputs, *held, *dims, **place, out=target)
    for side, (x, g, n) in enumerate(zip(rows, gradients, (heads, kv_heads))):
        if not n:
            assert out[side] is None and back[side] is None and back[2 + side] is None
            continue
        shape = (positions, n, dim)
        (y, y_bound), (dx, dx_bound), dw = reference(x.reshape(shape), weights[side], angle, g.reshape(shape))
        assert out[side].dtype == dtype
        within(download(out[side]).reshape(shape), y, y_bound, dtype)
        got = download(back[side]).reshape(positions, -1)
        if stacked:
            start = side * wide[0]
            got, block = got[:, start:start + wide[side]], got
            assert (block[:, wide[0] + wide[1]:] == 7.0).all()  # the other columns are left as they were
        within(got.reshape(shape), dx, dx_bound, dtype)
        if not normed:
            assert back[2 + side] is None
            continue
        expected, bound, terms = dw
        chain = positions * (heads + kv_heads) / 64 + 1100  # additions that a term can pass through
        assert (np.abs(download(back[2 + side]) - expected) <= bound + chain * UNIT * terms).all()


def test_gradients_agree_with_differences():
    """The recorded op: central differences of sum(y * c) in float64 at the
    kernel's inputs, along random directions."""
    rng = np.random.default_rng(5)
    batch, time, heads, kv_heads, dim = 2, 5, 4, 2, 16
    q, k = (rng.standard_normal((batch, time, n * dim)).astype(np.float32) for n in (heads, kv_heads))
    wq, wk = ((1 + 0.2 * rng.standard_normal(dim)).astype(np.float32) for _ in range(2))
    c = [rng.standard_normal(x.shape).astype(np.float32) for x in (q, k)]
    leaves = [Tensor(upload(x, "float32"), shape=x.shape, requires_grad=True) for x in (q, k, wq, wk)]
    y = qk_norm_rope(*leaves, heads, kv_heads, THETA, EPS, offset=3)
    for out, weight in zip(y, c):
        out.backward(Tensor(upload(weight, "float32"), shape=weight.shape))
    angle = (3 + np.arange(time))[None, :, None, None] * THETA ** (-np.arange(0, dim, 2) / dim)

    def value(parts):
        total = 0.0
        for x, w, weight in zip(parts[:2], parts[2:], c):
            rows = x.reshape(batch, time, -1, dim)
            total += (reference(rows, w, angle)[0] * weight.reshape(rows.shape)).sum()
        return total

    base = [x.astype(np.float64) for x in (q, k, wq, wk)]
    for i, leaf in enumerate(leaves):
        grad = download(leaf.grad.storage).reshape(base[i].shape)
        step = rng.standard_normal(base[i].shape)
        h = 1e-5
        moved = [value([b + (s * h * step if j == i else 0) for j, b in enumerate(base)]) for s in (1, -1)]
        slope = (moved[0] - moved[1]) / (2 * h)
        # the third derivative times h^2 / 6 is some 1e-9; fp32 gradients of a few hundred terms
        assert abs(slope - (grad * step).sum()) <= 1e-8 + 400 * UNIT * np.abs(grad * step).sum() + 1e-6


def test_weight_gradients_are_the_same_every_time():
    rng = np.random.default_rng(1)
    x, g = (upload(rng.standard_normal((400, 8 * 64)), "bfloat16") for _ in range(2))
    w = upload(np.ones(64), "float32")
    runs = [amd_lm.qk_norm_rope_backward(g, None, x, None, w, None, 4, 100, 8, 0, 64, THETA, EPS) for _ in range(3)]
    for run in runs[1:]:
        assert run[0].to_array() == runs[0][0].to_array() and run[2].to_array() == runs[0][2].to_array()


@pytest.mark.parametrize("batch,time", [(0, 5), (3, 0)])
def test_no_positions(batch, time):
    empty, w = amd.AMDStorage(0, "bfloat16"), upload(np.ones(8), "float32")
    dims = (batch, time, 2, 1, 8, THETA, EPS)
    out = amd_lm.qk_norm_rope(empty, empty, w, w, *dims)
    assert [x.size for x in out] == [0, 0]
    back = amd_lm.qk_norm_rope_backward(empty, empty, empty, empty, w, w, *dims)
    assert [x.size for x in back[:2]] == [0, 0]
    assert all((download(x) == 0).all() for x in back[2:])


@pytest.mark.parametrize("cast", [False, True])
def test_decoder_trains_with_normed_heads(cast):
    """Decoder(qk_norm=True): its loss's gradient along a direction of each
    norm weight against differences of the loss (fp32), and finite under autocast."""
    config = Config(vocab_size=64, n_layers=1, d_model=32, n_heads=4, n_kv_heads=2, d_ff=48, max_seq_len=16,
                    qk_norm=True)
    model = Decoder(config, seed=3)
    names = [n for n, _ in model.named_parameters()]
    assert "blocks.0.attn.q_norm.weight" in names
    assert sum(p.size for p in model.parameters()) == config.parameter_counts()["total_parameters"]
    rng = np.random.default_rng(2)
    tokens = rng.integers(0, 64, (2, 12)).tolist()
    if cast:
        with autocast():
            loss = model.loss(tokens)
        loss.backward()
        assert all(np.isfinite(download(p.grad.storage)).all() for p in model.parameters())
        return
    # larger weights, so that the loss moves with the norms
    for name, p in model.named_parameters():
        if name.endswith((".q.weight", ".k.weight", ".v.weight", ".out.weight", "embedding.weight")):
            amd.copy_into(p.storage, upload(rng.standard_normal(p.shape) * 0.4, "float32"))
    loss = model.loss(tokens)
    loss.backward()
    parameters = dict(model.named_parameters())
    for name in ("blocks.0.attn.q_norm.weight", "blocks.0.attn.k_norm.weight"):
        p = parameters[name]
        base, grad = download(p.storage).astype(np.float64), download(p.grad.storage)
        direction = np.sign(grad)
        losses = []
        for sign in (1, -1):
            amd.copy_into(p.storage, upload(base + sign * 0.02 * direction, "float32"))
            losses.append(float(model.loss(tokens, train=False).item()))
        amd.copy_into(p.storage, upload(base, "float32"))
        slope, expected = (losses[0] - losses[1]) / 0.04, np.abs(grad).sum()
        # each loss (about 5) is rounded to some 20 units of fp32: 6e-6 of slope here is 2 * 20 * 5 * 2^-24 / 0.04 = 3e-4;
        # the cubic term of a step of 2 % is of the order of 1e-3 of the slope
        assert abs(slope - expected) <= 3e-4 + 0.01 * expected


def test_checkpoint_keeps_the_norms(tmp_path):
    """A decoder with normed heads saved and loaded; one without refuses its files."""
    from qutai_amd.lm import load_checkpoint, save_checkpoint

    sizes = dict(vocab_size=40, n_layers=1, d_model=16, n_heads=2, n_kv_heads=1, d_ff=24, max_seq_len=8)
    model, other = (Decoder(Config(**sizes, qk_norm=True), seed=s) for s in (1, 2))
    weights = dict(model.named_parameters())
    amd.copy_into(weights["blocks.0.attn.q_norm.weight"].storage, upload(np.arange(8) + 0.5, "float32"))
    save_checkpoint(tmp_path / "saved", model)
    load_checkpoint(tmp_path / "saved", other)
    for name, p in other.named_parameters():
        assert p.storage.to_array() == weights[name].storage.to_array(), name
    with pytest.raises(ValueError):
        load_checkpoint(tmp_path / "saved", Decoder(Config(**sizes), seed=3))
