"""Decoder-only language model on the MI355X (src/qutai/lm/decoder.py:20-175).

Embedding (tied with the output head), ``n_layers`` pre-norm blocks (GQA
attention with RoPE, SwiGLU or top-k MoE FFN), a final RMSNorm, and the
chunked next-token loss.  Every op runs on the device through the HIP
kernels of ``qutai_amd.backends.amd_lm``: the training step reads nothing
back to the host.

Parameters are fp32; under ``autocast`` (matmul precision bfloat16) the
projections, attention and FFN run on bf16 activations while the residual
stream, norms and parameter gradients stay fp32, as in the reference.  A MoE
block stores each projection of all experts as one (experts, out, in) tensor:
``named_parameters`` names them ``ffn.experts.gate.weight`` etc.; expert e of
the reference's ``ffn.experts.{e}.gate.weight`` is row block e.
"""
from __future__ import annotations

from array import array
from bisect import bisect_left
from functools import partial
from itertools import chain
from random import Random

from ..backends import amd
from ..core.context import set_recording
from ..core.tensor import Tensor
from .config import Config
from ..nn.cache import QuantizedKVCache, unchanged_on_failure
from .packing import Packing
from .layers import Block, Projection, RMSNorm, backend, embed, linear, projection_loss, sample, scaled, unpack
from .recompute import checkpoint


def _int_array(values):
    """int64 array of host ids (C-level conversion; other numbers via int())."""
    values = list(values)
    try:
        return array("q", values)
    except TypeError:
        return array("q", (int(v) for v in values))


class Decoder:
    def __init__(self, config: Config, *, device="amd", dtype=None, seed=None):
        dtype = "float32" if dtype is None else dtype
        if device != "amd":
            raise ValueError("this Decoder runs on the amd device")
        if dtype != "float32":
            raise ValueError("decoder parameters on the amd device are float32 (bf16 activations via autocast)")
        self.config = config
        self.embedding = Projection(config.d_model, config.vocab_size, device=device, dtype=dtype, seed=seed)
        self.blocks = tuple(Block(config, device=device, dtype=dtype, seed=None if seed is None else seed + 1 + 100 * i)
                            for i in range(config.n_layers))
        self.norm = RMSNorm(config.d_model, config.norm_eps, device=device, dtype=dtype)
        self.last_lm_loss = None
        self.last_auxiliary_loss = None

    # ---- parameters (decoder.py:39-90) -------------------------------------------
    def named_parameters(self):
        result = [("embedding.weight", self.embedding.weight)]
        for i, block in enumerate(self.blocks):
            p = f"blocks.{i}."
            result += [(p + "attn_norm.weight", block.attn_norm.weight), (p + "ffn_norm.weight", block.ffn_norm.weight)]
            result += [(p + f"attn.{n}.weight", getattr(block.attn, n).weight) for n in ("q", "k", "v", "out")]
            if block.attn.q_norm is not None:
                result += [(p + f"attn.{n}.weight", getattr(block.attn, n).weight) for n in ("q_norm", "k_norm")]
            if block.is_moe:
                result.append((p + "ffn.router.weight", block.ffn.router.weight))
                result += [(p + "ffn.experts.gate.weight", block.ffn.w_gate), (p + "ffn.experts.up.weight", block.ffn.w_up),
                           (p + "ffn.experts.down.weight", block.ffn.w_down)]
            else:
                result += [(p + f"ffn.{n}.weight", getattr(block.ffn, n).weight) for n in ("gate", "up", "down")]
        result.append(("norm.weight", self.norm.weight))
        return tuple(result)

    def parameters(self):
        return tuple(dict.fromkeys(p for _, p in self.named_parameters()))

    def parameter_counts(self):
        return self.config.parameter_counts()

    # ---- forward (decoder.py:92-139) -----------------------------------------------
    def _tokens(self, tokens):
        rows = [row if isinstance(row, (list, tuple)) else list(row) for row in tokens]
        if not rows or any(len(row) != len(rows[0]) for row in rows) or not 1 <= len(rows[0]) <= self.config.max_seq_len:
            raise ValueError("tokens must be a non-empty 2-D batch no longer than max_seq_len")
        ids = _int_array(chain.from_iterable(rows))  # C-level loops: the ids feed every step
        if min(ids) < 0 or max(ids) >= self.config.vocab_size:
            raise ValueError("token id outside the vocabulary")
        return ids, (len(rows), len(rows[0]))

    def hidden(self, tokens, *, train=True):
        with set_recording(train):
            return self._hidden(tokens, train=train)

    def _hidden(self, tokens, *, train=True):
        return self._blocks(*self._tokens(tokens), train)

    def _blocks(self, ids, shape, train, packing=None):
        hidden = embed(ids, self.embedding.weight, shape)
        auxiliary = []
        for block in self.blocks:
            if train and self.config.activation_checkpointing:
                if block.is_moe:
                    function = partial(block.packed, packing=packing)
                    hidden, aux = unpack(checkpoint(function, hidden, parameters=block.parameters()), hidden.shape)
                else:
                    hidden = checkpoint(partial(block.hidden, packing=packing), hidden, parameters=block.parameters())
                    aux = Tensor(amd.full(1, 0.0, dtype=hidden.dtype), shape=())
            else:
                hidden, aux = block(hidden, packing)
            auxiliary.append(aux)
        total = auxiliary[0]
        for value in auxiliary[1:]:
            total = total + value.to(dtype=total.dtype)
        self.last_auxiliary_loss = scaled(total, 1 / self.config.n_layers)
        return self.norm(hidden)

    def __call__(self, tokens, *, train=True):
        """Logits (batch, time, vocab) of the tied head (decoder.py:134-139)."""
        with set_recording(train):
            return linear(self.hidden(tokens, train=train), self.embedding.weight)

    # ---- answering: new positions over quantised caches ----------------------------
    def caches(self, capacity=None, *, bits=8):
        """An empty QuantizedKVCache for each block (capacity: max_seq_len)."""
        capacity = self.config.max_seq_len if capacity is None else capacity
        return tuple(QuantizedKVCache(capacity, bits=bits) for _ in self.blocks)

    def decode(self, tokens, caches, counts=None):
        """Logits (batch, vocab) that follow the last of ``tokens`` (batch, new),
        the positions behind those that ``caches`` hold; of sequence b only the
        first counts[b] are there, at least one.  Nothing is recorded; a call
        that fails leaves the caches as they were."""
        ids, (batch, new) = self._tokens(tokens)
        caches = tuple(caches)
        counts = (new,) * batch if counts is None else tuple(counts)
        if len(caches) != len(self.blocks) or len(counts) != batch or any(type(n) is not int or not 1 <= n <= new for n in counts):
            raise ValueError("decode takes a cache for each block and a count of 1 to new positions for each sequence")
        if len({id(c) for c in caches}) != len(caches):
            raise ValueError("every block needs a cache of its own")
        held = caches[0].lengths or (0,) * batch
        if any((c.lengths or (0,) * batch) != held for c in caches) or len(held) != batch:
            raise ValueError("the caches hold other sequences than the tokens'")
        limit = min(self.config.max_seq_len, *(c.capacity for c in caches))
        if any(n + m > limit for n, m in zip(held, counts)):
            raise ValueError("the positions exceed max_seq_len or the caches' capacity")
        with set_recording(False), unchanged_on_failure(*caches):
            hidden = embed(ids, self.embedding.weight, (batch, new))
            for block, cache in zip(self.blocks, caches):
                hidden = block.decode(hidden, cache, None if min(counts) == new else counts)
            if new > 1:  # the rows that a token follows
                last = array("q", (b * new + n - 1 for b, n in enumerate(counts)))
                width = self.config.d_model
                rows = backend(hidden).embedding(hidden.storage, last, width)
                hidden = Tensor(rows, shape=(batch, 1, width))
            hidden = self.norm(hidden)
            return linear(Tensor(hidden.storage, shape=(batch, self.config.d_model)), self.embedding.weight)

    def generate(self, prompts, count, *, seed=None, bits=8, **filters):
        """``count`` tokens behind each prompt (lists of ids of any lengths), one
        list for each: every step's logits are sampled (``filters``:
        temperature, top_k, top_p, min_p) with numbers of Random(seed), one per
        sequence and step, keys and values cached in codes of ``bits``."""
        prompts = [list(p) for p in prompts]
        if type(count) is not int or count < 0 or not prompts or not all(prompts):
            raise ValueError("generate takes prompts of one token at least and a number of tokens")
        counts = [len(p) for p in prompts]
        total = max(counts) + max(0, count - 1)
        if total > self.config.max_seq_len:
            raise ValueError("prompt and generated tokens exceed max_seq_len")
        random, made = Random(seed), [[] for _ in prompts]
        caches = self.caches(total, bits=bits)
        tokens = [p + [0] * (max(counts) - len(p)) for p in prompts]
        for _ in range(count):
            logits = self.decode(tokens, caches, counts)
            chosen, _ = sample(logits, [random.random() for _ in prompts], **filters)
            if min(chosen) < 0:
                raise RuntimeError("a row of logits holds no number that a token can be sampled from")
            for row, token in zip(made, chosen):
                row.append(token)
            tokens, counts = [[token] for token in chosen], [1] * len(prompts)
        return made

    # ---- loss (decoder.py:141-175) -------------------------------------------------
    def loss(self, tokens, labels=None, *, train=True, chunk_size=128):
        if chunk_size <= 0:
            raise ValueError("chunk_size must be positive")
        _, shape = self._tokens(tokens)
        if shape[1] < 2:
            raise ValueError("next-token training needs at least two positions")
        label_rows = self._labels(tokens if labels is None else labels, [shape[1]] * shape[0])
        with set_recording(train):
            prepared = backend(self.embedding.weight).prepare_labels(
                _int_array(chain.from_iterable(row[1:] for row in label_rows)))
            hidden = self.hidden(tokens, train=train)
            self.last_lm_loss = projection_loss(hidden, self.embedding.weight, label_rows, chunk_size,
                                                prepared_labels=prepared)
            aux = self.last_auxiliary_loss.to(dtype=self.last_lm_loss.dtype)
            return self.last_lm_loss + scaled(aux, self.config.aux_loss_coef)

    def _labels(self, labels, lengths):
        """The labels as rows of these lengths; ValueError where they are not, or
        hold anything but vocabulary ids and -100."""
        rows = [row if isinstance(row, (list, tuple)) else list(row) for row in labels]
        if [len(row) for row in rows] != list(lengths):
            raise ValueError("labels must have the shape of tokens")
        ordered = sorted(_int_array(chain.from_iterable(rows)))
        first = bisect_left(ordered, -99)  # first label above the ignore id
        if ordered[0] < -100 or ordered[-1] >= self.config.vocab_size or (first < len(ordered) and ordered[first] < 0):
            raise ValueError("labels must be vocabulary ids or -100")
        return rows

    def loss_packed(self, sequences, labels=None, *, train=True, chunk_size=128):
        """``loss`` of sequences of different lengths (lists of ids, each no longer
        than max_seq_len), which lie one behind the other in one row of tokens: no
        padding, no token sees another sequence, and positions start at 0 in each.
        The mean runs over the predictions of all sequences (a sequence's last token
        predicts nothing); labels have the sequences' shape, -100 is ignored.  Under
        autocast attention rounds probabilities to bf16 (amd_lm.attention_packed), where
        that of ``loss`` does so for heads of 64 channels only."""
        if chunk_size <= 0:
            raise ValueError("chunk_size must be positive")
        rows = [row if isinstance(row, (list, tuple)) else list(row) for row in sequences]
        if not rows or any(not 1 <= len(row) <= self.config.max_seq_len for row in rows):
            raise ValueError("packed sequences hold one token at least and no more than max_seq_len")
        if sum(map(len, rows)) < 2:
            raise ValueError("next-token training needs at least two positions")
        ids = _int_array(chain.from_iterable(rows))
        if min(ids) < 0 or max(ids) >= self.config.vocab_size:
            raise ValueError("token id outside the vocabulary")
        label_rows = self._labels(rows if labels is None else labels, map(len, rows))
        # the token before a sequence's first predicts nothing
        targets = [list(chain.from_iterable((-100, *row[1:]) for row in label_rows))]
        packing = Packing(map(len, rows))
        with set_recording(train):
            prepared = backend(self.embedding.weight).prepare_labels(_int_array(targets[0][1:]))
            hidden = self._blocks(ids, (1, packing.total), train, packing)
            self.last_lm_loss = projection_loss(hidden, self.embedding.weight, targets, chunk_size,
                                                prepared_labels=prepared)
            aux = self.last_auxiliary_loss.to(dtype=self.last_lm_loss.dtype)
            return self.last_lm_loss + scaled(aux, self.config.aux_loss_coef)
