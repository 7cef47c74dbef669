"""A training step over packed documents: Decoder.loss_packed, its gradients and
AdamW, against the same documents one by one; with norms of heads, other rotary
positions, experts, recomputation and mixed precision; and answers of a model
whose positions are not the reference's."""
import numpy as np
import pytest

from qutai_amd.lm import Config, Decoder, Packing, Rotary, autocast
from qutai_amd.optim import AdamW
from tests.helpers import download

pytestmark = pytest.mark.gpu

SMALL = dict(vocab_size=96, n_layers=2, d_model=64, n_heads=4, n_kv_heads=2, d_ff=96, max_seq_len=64,
             activation_checkpointing=False)
DOCUMENTS = [[5, 7, 9, 11, 2], [3], [1, 2], [90 - i for i in range(40)], [8] * 17]
VARIANTS = {
    "plain": {}, "checkpointed": dict(activation_checkpointing=True), "normed": dict(qk_norm=True),
    "half": dict(rope_layout="half", rope_scaling={"kind": "linear", "factor": 2.0}),
    "part": dict(rope_dim=8, rope_layout="half", qk_norm=True,
                 rope_scaling={"kind": "parts", "factor": 4.0, "original_length": 16}),
    "experts": dict(ffn_type="moe", n_experts=4, top_k=2, d_expert=48, aux_loss_coef=0.0, activation_checkpointing=True),
}


def gradients(model):
    return {n: download(p.grad.storage).astype(np.float64) for n, p in model.named_parameters()}


def one_by_one(model, documents):
    """(loss, gradients): the mean over all predictions, a document at a time."""
    count = sum(len(d) - 1 for d in documents)
    total, sums = 0.0, {}
    for d in documents:
        if len(d) < 2:
            continue
        for p in model.parameters():
            p.zero_grad()
        loss = model.loss([d])
        loss.backward()
        share = (len(d) - 1) / count
        total += share * loss.item()
        for n, g in gradients(model).items():
            sums[n] = sums.get(n, 0) + share * g
    return total, sums


@pytest.mark.parametrize("variant", VARIANTS)
def test_packed_documents_are_the_documents(variant):
    model = Decoder(Config(**{**SMALL, **VARIANTS[variant]}), seed=1)
    expected, sums = one_by_one(model, DOCUMENTS)
    for p in model.parameters():
        p.zero_grad()
    loss = model.loss_packed(DOCUMENTS, chunk_size=16)
    loss.backward()
    assert abs(loss.item() - expected) <= 1e-5 * expected
    for name, g in gradients(model).items():
        # sums of fp32 roundings along two different orders: the bar of the decoder's own tests
        assert np.abs(g - sums[name]).max() <= 2e-5 * (1 + np.abs(sums[name]).max()), name


@pytest.mark.parametrize("variant", ["plain", "normed", "half", "part"])
def test_mixed_precision(variant):
    config = Config(**{**SMALL, "d_model": 256, **VARIANTS[variant]})
    model = Decoder(config, seed=2)
    with autocast():
        expected, sums = one_by_one(model, DOCUMENTS)
        for p in model.parameters():
            p.zero_grad()
        loss = model.loss_packed(DOCUMENTS)
        loss.backward()
    assert abs(loss.item() - expected) <= 1e-2 * expected
    for name, g in gradients(model).items():  # bf16's bar of the decoder's own tests
        assert np.linalg.norm(g - sums[name]) <= 3e-2 * np.linalg.norm(sums[name]), name


@pytest.mark.parametrize("variant", ["half", "part"])
def test_other_rotations_in_rectangles_and_answers(variant):
    """loss over rectangles and cached decoding turn heads as loss_packed does."""
    for mixed in (False, True):
        model = Decoder(Config(**{**SMALL, "d_model": 256, **VARIANTS[variant]}), seed=3)
        rows = [[1, 2, 3, 4, 5, 6], [9, 8, 7, 6, 5, 4]]
        with autocast(mixed):
            packed, loss = model.loss_packed(rows).item(), model.loss(rows).item()
            assert abs(packed - loss) <= (1e-2 if mixed else 1e-5) * loss
            logits = download(model(rows, train=False).storage).reshape(2, 6, -1)
            caches = model.caches(8)
            model.decode([r[:4] for r in rows], caches)
            model.decode([r[4:5] for r in rows], caches)
            last = download(model.decode([r[5:] for r in rows], caches).storage).reshape(2, -1)
        # keys and values held in 8 bits: the bar of the decoder's cached decoding
        assert np.linalg.norm(last - logits[:, 5]) <= 5e-2 * np.linalg.norm(logits[:, 5])


@pytest.mark.parametrize("bits", [8, 32])
def test_training_steps(bits):
    """Losses over packed documents, backward and AdamW in a row: every parameter
    moves, the state of another process goes on with the same bits."""
    runs = []
    for _ in range(2):
        model = Decoder(Config(**SMALL), seed=5)
        optimizer = AdamW(model.parameters(), lr=3e-3, bits=bits, max_norm=1.0)
        start = [download(p.storage) for p in model.parameters()]
        for step in range(3):
            optimizer.zero_grad()
            model.loss_packed(DOCUMENTS[step % 2:]).backward()
            optimizer.step()
            assert np.isfinite(optimizer.norm())
        runs.append([download(p.storage) for p in model.parameters()])
        assert all((a != b).any() for a, b in zip(start, runs[-1]))
    assert all(np.array_equal(a, b) for a, b in zip(*runs))


def test_labels_of_packed_documents():
    model = Decoder(Config(**SMALL), seed=7)
    labels = [list(d) for d in DOCUMENTS]
    labels[3][1:30] = [-100] * 29
    labels[0][0] = 50  # no token predicts a document's first
    loss = model.loss_packed(DOCUMENTS, labels).item()
    count = total = 0
    for d, l in zip(DOCUMENTS, labels):
        n = sum(x != -100 for x in l[1:])
        if n:
            total += n * model.loss([d], [l]).item()
            count += n
    assert abs(loss - total / count) <= 1e-5 * loss


def test_checkpoints_keep_the_rotation(tmp_path):
    """A model whose positions are not the reference's is saved and read back."""
    from qutai_amd.lm import load_checkpoint, save_checkpoint

    config = Config(**{**SMALL, **VARIANTS["part"]})
    model = Decoder(config, seed=11)
    model.loss_packed(DOCUMENTS).backward()
    save_checkpoint(tmp_path, model)
    other = Decoder(Config(**config.to_dict()), seed=12)
    load_checkpoint(tmp_path, other)
    assert model.loss_packed(DOCUMENTS).item() == other.loss_packed(DOCUMENTS).item()
    with pytest.raises(ValueError):  # another rotation is another model
        load_checkpoint(tmp_path, Decoder(Config(**SMALL, qk_norm=True), seed=12))


def test_evaluation_records_nothing():
    model = Decoder(Config(**SMALL), seed=13)
    loss = model.loss_packed(DOCUMENTS, train=False)
    assert not loss.requires_grad
