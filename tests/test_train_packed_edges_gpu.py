"""Decoder.loss_packed where nothing or little is predicted, at the longest document, and
with arguments that are read once."""
import numpy as np
import pytest

from qutai_amd.lm import Config, Decoder, autocast
from tests.helpers import download

pytestmark = pytest.mark.gpu

SMALL = dict(vocab_size=96, n_layers=2, d_model=64, n_heads=4, n_kv_heads=2, d_ff=96, max_seq_len=40, activation_checkpointing=False)


@pytest.mark.parametrize("mixed", [False, True])
@pytest.mark.parametrize("labels", [None, [[7], [-100], [9]]])
def test_documents_of_one_token_predict_nothing(labels, mixed):
    """A document's last token predicts nothing: the loss is 0, and so is every gradient."""
    model = Decoder(Config(**{**SMALL, "d_model": 256 if mixed else 64}), seed=1)
    with autocast(mixed):
        loss = model.loss_packed([[3], [5], [9]], labels)
        loss.backward()
    assert loss.item() == 0.0
    assert all(not download(p.grad.storage).any() for p in model.parameters())


@pytest.mark.parametrize("change", [{}, dict(rope_layout="half"), dict(qk_norm=True)])
def test_the_shortest_and_the_longest_document(change):
    """Two tokens, and as many as the model takes, alone and one behind the other."""
    model = Decoder(Config(**SMALL, **change), seed=2)
    documents = [[4, 8], [(7 * i) % 96 for i in range(40)]]
    alone = [model.loss_packed([d], train=False).item() for d in documents]
    for d, loss in zip(documents, alone):
        assert abs(model.loss([d], train=False).item() - loss) <= 1e-5 * loss
    both = model.loss_packed(documents, train=False).item()
    assert abs(both - (alone[0] + 39 * alone[1]) / 40) <= 1e-5 * both


def test_sequences_and_labels_of_any_kind_are_read_once():
    model = Decoder(Config(**SMALL), seed=3)
    documents = [[1, 2, 3], [4, 5]]
    expected = model.loss_packed(documents, train=False).item()
    given = (iter(d) for d in documents), (np.array(d) for d in documents)
    assert model.loss_packed(given[0], train=False).item() == expected
    assert model.loss_packed([tuple(d) for d in documents], given[1], train=False).item() == expected


@pytest.mark.parametrize("sequences,labels", [
    ([], None), ([[]], None), ([[1, 2], []], None), ([[1]], None), ([list(range(41))], None), ([[1, 96]], None), ([[1, -1]], None),
    ([[1, 2]], [[1]]), ([[1, 2]], [[1, 2], [3]]), ([[1, 2]], [[1, 96]]), ([[1, 2]], [[1, -2]]), ([[1, 2]], [])])
def test_refusals(sequences, labels):
    model = Decoder(Config(**SMALL), seed=4)
    with pytest.raises(ValueError):
        model.loss_packed(sequences, labels)
