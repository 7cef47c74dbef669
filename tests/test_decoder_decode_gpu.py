"""Answering with a Decoder: cached decoding over quantised caches (normed and
rotated heads, codes written and read by attention, sampled tokens together)
against a float64 forward pass that reads the values the caches hold."""
import numpy as np
import pytest

from qutai_amd import Tensor
from qutai_amd.backends import amd, amd_lm
from qutai_amd.lm import Config, Decoder, autocast, sample
from qutai_amd.nn import MultiHeadAttention, QuantizedKVCache
from tests.helpers import download, stored, upload
from tests.test_cache_quantized_gpu import held

pytestmark = pytest.mark.gpu


def build(qk_norm, ffn="dense", width=32, heads=4, kv_heads=2, layers=2):
    config = Config(vocab_size=61, n_layers=layers, d_model=width, n_heads=heads, n_kv_heads=kv_heads, d_ff=40, max_seq_len=48,
                    ffn_type=ffn, n_experts=4, top_k=2, d_expert=24, qk_norm=qk_norm)
    model = Decoder(config, seed=1)
    rng = np.random.default_rng(0)
    for name, p in model.named_parameters():
        x = rng.standard_normal(p.shape) * 0.3
        amd.copy_into(p.storage, upload(1 + x / 3 if "norm" in name else x, "float32"))
    return model


def norm(x, w, eps):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w


def turned(x, at, theta):
    angle = at[:, None, None] * theta ** (-np.arange(0, x.shape[-1], 2) / x.shape[-1])
    out = np.empty_like(x)
    out[..., 0::2] = x[..., 0::2] * np.cos(angle) - x[..., 1::2] * np.sin(angle)
    out[..., 1::2] = x[..., 0::2] * np.sin(angle) + x[..., 1::2] * np.cos(angle)
    return out


class Reference:
    """One sequence's new positions in float64, over the values that the caches hold."""

    def __init__(self, model):
        self.c = model.config
        self.p = {n: download(p.storage).astype(np.float64).reshape(p.shape) for n, p in model.named_parameters()}

    def logits(self, tokens, start, caches, sequence, bits, rounded=None):
        """``rounded``: applied where autocast stores bf16 (inputs and weights of
        every product, and its result; the caches' values are as they are)."""
        c, p = self.c, self.p
        r = rounded or (lambda x: x)
        x = p["embedding.weight"][tokens]
        at = start + np.arange(len(tokens))
        head, group = c.d_model // c.n_heads, c.n_heads // c.n_kv_heads
        for i, cache in enumerate(caches):
            a = f"blocks.{i}.attn."
            y = r(norm(x, p[f"blocks.{i}.attn_norm.weight"], c.norm_eps))
            q, k, v = (r(y @ r(p[a + n + ".weight"]).T) for n in "qkv")
            q, k, v = (z.reshape(len(tokens), -1, head) for z in (q, k, v))
            if c.qk_norm:
                q, k = norm(q, p[a + "q_norm.weight"], c.norm_eps), norm(k, p[a + "k_norm.weight"], c.norm_eps)
            q, k = r(turned(q, at, c.rope_theta)), r(turned(k, at, c.rope_theta))
            keys, values = (download(z.storage).reshape(z.shape)[sequence].astype(np.float64) for z in cache.read())
            for got, fresh in ((keys, k), (values, v)) if rounded is None else ():
                # a code's half step, and a flip where the fp32 value lies on the other side of a border
                exact = fresh.transpose(1, 0, 2)
                step = np.abs(exact).max() * 1.01 / (127 if bits == 8 else 7)
                assert np.abs(got[:, at] - exact).max() <= 0.51 * step
            mixed = np.empty_like(q)
            for h in range(c.n_heads):
                s = q[:, h] @ keys[h // group, :at[-1] + 1].T / head ** 0.5
                s[np.arange(at[-1] + 1)[None] > at[:, None]] = -np.inf
                w = np.exp(s - s.max(1, keepdims=True))
                mixed[:, h] = w / w.sum(1, keepdims=True) @ values[h // group, :at[-1] + 1]
            x = x + r(r(mixed).reshape(len(tokens), -1) @ r(p[a + "out.weight"]).T)
            y = r(norm(x, p[f"blocks.{i}.ffn_norm.weight"], c.norm_eps))
            f = f"blocks.{i}.ffn."
            gate, up = r(y @ r(p[f + "gate.weight"]).T), r(y @ r(p[f + "up.weight"]).T)
            x = x + r(r(r(gate / (1 + np.exp(-gate))) * up) @ r(p[f + "down.weight"]).T)
        return r(r(norm(x, p["norm.weight"], c.norm_eps)[-1]) @ r(p["embedding.weight"]).T)


@pytest.mark.parametrize("qk_norm,bits,ragged", [(True, 8, True), (True, 4, False), (False, 8, True), (False, 8, False)])
def test_cached_logits_match_float64(qk_norm, bits, ragged):
    model = build(qk_norm)
    reference, caches = Reference(model), model.caches(bits=bits)
    rng = np.random.default_rng(3)
    lengths = [0, 0, 0]
    for new in (7, 1, 3, 1):
        tokens = rng.integers(0, 61, (3, new)).tolist()
        counts = [max(1, new - 2 * b) for b in range(3)] if ragged else None
        logits = model.decode(tokens, caches, counts)
        assert logits.shape == (3, 61) and not logits.requires_grad
        got = download(logits.storage).reshape(3, 61)
        for b in range(3):
            n = counts[b] if ragged else new
            expected = reference.logits(tokens[b][:n], lengths[b], caches, b, bits)
            # sums of 32 to 40 fp32 products through two blocks: some thousand roundings of values of this size
            assert np.abs(got[b] - expected).max() <= 2000 * 2.0 ** -24 * np.abs(expected).max()
            lengths[b] += n
        assert all(c.lengths == tuple(lengths) for c in caches)


def test_autocast_decoding_rounds_as_bf16_does():
    """bf16 activations (one projection product, its columns read in place)
    against float64 over the values the caches hold.  How far the storage's
    roundings may carry is seen from the same pass with them: another order of
    sums gives roundings of the same sizes, so three times its own distance."""
    model = build(True, width=64, heads=4, kv_heads=2)
    reference, caches, rng = Reference(model), model.caches(), np.random.default_rng(5)
    start = 0
    for new in (6, 1, 1):
        tokens = rng.integers(0, 61, (2, new)).tolist()
        with autocast():
            got = download(model.decode(tokens, caches).storage).reshape(2, 61)
        for b in range(2):
            exact, low = (reference.logits(tokens[b], start, caches, b, 8, r)
                          for r in (lambda x: x, lambda x: stored(x, "bfloat16")))
            assert np.linalg.norm(got[b] - exact) <= 3 * np.linalg.norm(low - exact)
        start += new


@pytest.mark.parametrize("qk_norm,ffn", [(True, "dense"), (False, "moe")])
def test_decoding_agrees_with_the_whole_forward_pass(qk_norm, ffn):
    """Logits of cached decoding against the uncached model on the same tokens:
    apart by what 8-bit keys and values are off."""
    model = build(qk_norm, ffn)
    tokens = np.random.default_rng(8).integers(0, 61, (2, 12)).tolist()
    whole = download(model(tokens, train=False).storage).reshape(2, 12, 61)
    caches = model.caches()
    model.decode([row[:9] for row in tokens], caches)
    for t in (9, 10, 11):
        got = download(model.decode([[row[t]] for row in tokens], caches).storage).reshape(2, 61)
        # half a step of 1/127 of a row's largest value in each key and value, and through two blocks
        assert np.linalg.norm(got - whole[:, t]) <= 0.05 * np.linalg.norm(whole[:, t])


def test_generate_samples_what_decode_gives():
    from random import Random

    model = build(True)
    prompts, filters = [[3, 4, 5, 6], [7], [8, 9]], dict(temperature=0.8, top_k=20, top_p=0.9)
    made = model.generate(prompts, 6, seed=11, **filters)
    assert [len(row) for row in made] == [6, 6, 6] and all(0 <= t < 61 for row in made for t in row)
    assert made == model.generate(prompts, 6, seed=11, **filters)
    random, caches = Random(11), model.caches(9)
    tokens, counts = [p + [0] * (4 - len(p)) for p in prompts], [4, 1, 2]
    for step in range(6):
        logits = model.decode(tokens, caches, counts)
        chosen, probabilities = sample(logits, [random.random() for _ in prompts], **filters)
        assert chosen == [row[step] for row in made] and all(0 < x <= 1 for x in probabilities)
        tokens, counts = [[t] for t in chosen], [1, 1, 1]
    greedy = model.generate(prompts, 3, temperature=0.0)
    logits = model.decode([p + [0] * (4 - len(p)) for p in prompts], model.caches(), [4, 1, 2])
    assert [row[0] for row in greedy] == download(logits.storage).reshape(3, 61).argmax(1).tolist()
    assert model.generate([[1]], 0) == [[]]


@pytest.mark.parametrize("failing", [0, 1])
def test_a_step_that_failed_can_be_made_again(failing, monkeypatch):
    """The attention of a block raises: the caches hold what they did, and the
    same call then gives the logits of a run without the failure."""
    model, rng = build(True), np.random.default_rng(7)
    steps = [rng.integers(0, 61, (2, new)).tolist() for new in (4, 1)]
    whole = model.caches()
    expected = [model.decode(tokens, whole).storage.to_array() for tokens in steps]
    caches, attention = model.caches(), amd_lm.attention_quantized
    for tokens, logits in zip(steps, expected):
        held, calls = [(c.lengths, c.codes) for c in caches], []

        def fail(*arguments, **options):
            calls.append(None)
            if len(calls) > failing:
                raise RuntimeError("no memory left")
            return attention(*arguments, **options)

        with monkeypatch.context() as patch:
            patch.setattr(amd_lm, "attention_quantized", fail)
            with pytest.raises(RuntimeError):
                model.decode(tokens, caches)
        assert [(c.lengths, c.codes) for c in caches] == held
        assert model.decode(tokens, caches).storage.to_array() == logits


def test_layers_that_fail_append_nothing(monkeypatch):
    layer, heads = build(True, layers=1).blocks[0].attn, MultiHeadAttention(32, 4, causal=True, seed=1)
    x = Tensor(upload(np.random.default_rng(2).standard_normal((2, 3, 32)), "float32"), shape=(2, 3, 32))
    calls = (lambda cache: layer.decode(x, cache), lambda cache: heads(x, cache=cache))

    def fail(*arguments, **options):
        raise RuntimeError("no memory left")

    for call in calls:
        small = QuantizedKVCache(2)
        with pytest.raises(ValueError):
            call(small)  # too many positions: no batch or heads are settled
        assert small.codes is None and small.lengths == ()
        cache, whole = QuantizedKVCache(8), QuantizedKVCache(8)
        expected = [call(whole).storage.to_array() for _ in range(2)]
        for held, result in zip(((), (3, 3)), expected):
            with monkeypatch.context() as patch:
                patch.setattr(amd_lm, "attention_quantized", fail)
                with pytest.raises(RuntimeError):
                    call(cache)
            assert cache.lengths == held
            assert call(cache).storage.to_array() == result


@pytest.mark.parametrize("cast", [False, True])
@pytest.mark.parametrize("ffn", ["dense", "moe"])
def test_decoding_layers_record_nothing(ffn, cast):
    """GQA.decode and Block.decode called by themselves, with parameters and an
    input that require gradients; recording is on again behind them."""
    from contextlib import nullcontext

    block = build(True, ffn, layers=1).blocks[0]
    rng = np.random.default_rng(2)
    with autocast() if cast else nullcontext():
        for layer in (block.attn, block):
            x = Tensor(upload(rng.standard_normal((2, 3, 32)), "float32"), shape=(2, 3, 32), requires_grad=True)
            cache = QuantizedKVCache(8)
            y = layer.decode(x, cache)
            assert cache.lengths == (3, 3) and not y.requires_grad and y.parents == () and y.backward_rule is None
            attended = cache.attend(Tensor(upload(rng.standard_normal((2, 3, 4, 8)), "float32"), shape=(2, 3, 4, 8),
                                           requires_grad=True))
            assert not attended.requires_grad
            assert block.attn_norm(x).requires_grad


def test_refusals():
    model = build(True)
    caches = model.caches()
    for tokens, given, counts in (([[1, 2]], caches[:1], None), ([[1, 2]], caches, [3]), ([[1, 2]], caches, [0]),
                                  ([[1, 2]], caches, [1, 1]), ([[61]], caches, None), ([[1] * 49], caches, None)):
        with pytest.raises(ValueError):
            model.decode(tokens, given, counts)
    model.decode([[1, 2]], caches)
    for tokens in ([[1], [2]], [[1] * 47]):
        with pytest.raises(ValueError):
            model.decode(tokens, caches)
    for prompts, count in (([], 1), ([[]], 1), ([[1]], -1), ([[1] * 40], 10)):
        with pytest.raises(ValueError):
            model.generate(prompts, count)
    logits = model.decode([[1]], model.caches())
    with pytest.raises(ValueError):
        sample(logits, [0.5, 0.5])


def test_quantised_values_are_those_of_the_keys():
    """What a block caches is its normed and rotated keys' and its values' codes."""
    model = build(True, layers=1)
    caches = model.caches()
    model.decode([[5, 6, 7]], caches)
    keys, values = (download(x.storage).reshape(x.shape) for x in caches[0].read())
    again = [held(x.transpose(0, 2, 1, 3), 8).transpose(0, 2, 1, 3) for x in (keys, values)]
    # what the codes stand for lies on the codes' own grid: quantised again it moves by half a step at most
    for x, y in zip((keys, values), again):
        assert np.abs(x - y).max() <= 0.51 * np.abs(x).max() / 126


@pytest.mark.parametrize("qk_norm,bits", [(True, 8), (True, 4), (False, 8), (False, 4)])
def test_the_first_block_caches_the_codes_of_its_keys_and_values(qk_norm, bits):
    """What the first block's cache holds against the definition's codes of its
    normed and rotated keys and of its values, computed in float64 from the
    embedding's rows.  The kernel's fp32 keys and values are 34 roundings of 2^-24
    off at most, of sums some five times a row's largest value: 0.003 of a step of
    1/127 on either side of a border, so that some 0.3% of the codes (and, with a
    scale's 2^-8, as many scales) may be the next one's."""
    model = build(qk_norm)
    c, p = model.config, Reference(model).p
    rng, caches = np.random.default_rng(4), model.caches(bits=bits)
    kept = [[] for _ in range(3)]
    for counts in ((25, 9, 17), (1, 1, 1), (13, 14, 2)):
        tokens = rng.integers(0, 61, (3, max(counts))).tolist()
        model.decode(tokens, caches, counts)
        for row, new, n in zip(kept, tokens, counts):
            row += new[:n]
    read = [download(x.storage).reshape(x.shape) for x in caches[0].read()]
    changed = total = 0
    for b, tokens in enumerate(kept):
        y = norm(p["embedding.weight"][tokens], p["blocks.0.attn_norm.weight"], c.norm_eps)
        k, v = ((y @ p[f"blocks.0.attn.{n}.weight"].T).reshape(len(tokens), c.n_kv_heads, -1) for n in "kv")
        if qk_norm:
            k = norm(k, p["blocks.0.attn.k_norm.weight"], c.norm_eps)
        k = turned(k, np.arange(len(tokens)), c.rope_theta)
        for got, x in zip(read, (k, v)):
            got, expected = got[b, :, :len(tokens)].transpose(1, 0, 2), held(x, bits)
            # one step of a scale that is 2^-7 too large at most
            step = np.abs(x).max(-1, keepdims=True) * (1 + 2.0 ** -6) / (127 if bits == 8 else 7)
            assert (np.abs(got - expected) <= step).all()
            changed, total = changed + (got != expected).sum(), total + x.size
    assert changed <= 0.02 * total
