"""GQA with a Rotary on the bf16 path: what it sends, and what it computes, against its
steps one by one."""
import numpy as np
import pytest

from qutai_amd import Tensor
from qutai_amd.backends import amd, amd_lm
from qutai_amd.lm import GQA, Config, Packing, Rotary, autocast
from tests.helpers import download, normal, upload

pytestmark = pytest.mark.gpu

HEADS, KV_HEADS, WIDTH = 4, 2, 256


def calls_of(monkeypatch, function):
    """(the result, names of the library calls)."""
    runtime, names = amd.get_runtime(), []
    send = type(runtime).call

    def noted(name, *arguments, **options):
        names.append(name)
        return send(runtime, name, *arguments, **options)

    monkeypatch.setattr(runtime, "call", noted)
    result = function()
    monkeypatch.undo()
    return result, names


@pytest.mark.parametrize("qk_norm", [False, True])
@pytest.mark.parametrize("packed", [False, True])
def test_turned_heads_take_one_launch_and_no_copies(monkeypatch, qk_norm, packed):
    """One rotation for both sides; without a packing the values' columns alone are copied
    out of the product, with one nothing is."""
    config = Config(d_model=WIDTH, n_heads=HEADS, n_kv_heads=KV_HEADS, qk_norm=qk_norm, rope_layout="half",
                    rope_scaling={"kind": "linear", "factor": 2.0})
    gqa = GQA(config, device="amd", seed=3)
    batch, time = (1, 48) if packed else (2, 24)
    packing = Packing([20, 1, 27]) if packed else None
    x = Tensor(upload(normal(1, batch * time * WIDTH), "float32"), shape=(batch, time, WIDTH))
    with autocast():
        gqa(x, packing)  # tables and workspaces are there
        y, names = calls_of(monkeypatch, lambda: gqa(x, packing))
    assert names.count("qutai_amd_rotary") == 1
    assert names.count("qutai_amd_qk_norm_rope") == qk_norm
    assert names.count("qutai_amd_strided_copy") == (0 if packed else 1)

    # the same steps on their own
    dq, dkv, head = WIDTH, WIDTH * KV_HEADS // HEADS, WIDTH // HEADS
    rows = batch * time
    ws = amd.AMDStorage((dq + 2 * dkv) * WIDTH, "bfloat16")
    for w, start in ((gqa.q.weight, 0), (gqa.k.weight, dq), (gqa.v.weight, dq + dkv)):
        amd.cast_into(amd.view(ws, start * WIDTH, w.size), w.storage)
    xs = amd.AMDStorage(x.size, "bfloat16")
    amd.cast_into(xs, x.storage)
    qkv = amd_lm.gemm(xs, ws, rows, WIDTH, dq + 2 * dkv, transpose_right=True, out_dtype="bfloat16")
    q, k, v = (amd_lm.copy_rows(qkv, rows, n, column=c, row=dq + 2 * dkv) for n, c in ((dq, 0), (dkv, dq), (dkv, dq + dkv)))
    if qk_norm:
        q, k = amd_lm.qk_norm_rope(q, k, gqa.q_norm.weight.storage, gqa.k_norm.weight.storage, rows, 1, HEADS, KV_HEADS, head,
                                   config.rope_theta, config.norm_eps)
    turns = Rotary(head, config.rope_theta, layout="half", scaling={"kind": "linear", "factor": 2.0})
    q, k = amd_lm.rotary(q, k, turns, batch, time, HEADS, KV_HEADS, head, positions=packing.positions if packed else None)
    if packed:
        out, _ = amd_lm.attention_packed(q, k, v, packing, HEADS, KV_HEADS, head)
    else:
        out, _ = amd_lm.attention(q, k, v, batch, time, HEADS, KV_HEADS, head)
    with autocast():
        expected = gqa.out(Tensor(out, shape=(batch, time, WIDTH)))
    assert np.array_equal(download(y.storage), download(expected.storage))
