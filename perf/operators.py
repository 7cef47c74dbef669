"""The operators of a decoder that answers, as timed cases.

A case is a dict of plain values; its ``kind`` names one of the classes below:
norms of queries and keys per head with their position rotation (``qk``), a
key and value cache quantised as it is written and read back (``copy``),
attention of new positions over that cache (``attend``), and tokens sampled
from logits (``sample``).  Sizes are those of this repository's ``Config``
defaults (16 heads of 64 with 4 kv heads, vocabulary 32768, sequences of 1024)
and generic ones (32 heads of 128 with 8 kv heads, caches of thousands of
positions); odd ones are mixed in by ``draw``.

``prepare`` draws the inputs on the GPU from the seed.  Where ``own`` is false
``run`` computes an operator from elementary torch operations in 32 bits (64
for angles, quantised codes and sampling weights, where a value next to a
border would change the result); where it is true it calls the framework,
which is then given the same values as its own storages.  ``exact`` computes
the outputs in 64 bits from the operators' definitions.
"""
from __future__ import annotations

from math import exp, log

import torch

own = False

TORCH = {"float32": torch.float32, "bfloat16": torch.bfloat16}
BYTES = {"float32": 4, "bfloat16": 2}
THETA, EPS = 10000.0, 1e-6


# ---- between torch and the framework's storages -----------------------------------

RAW = {"float32": ("<f4", torch.float32), "bfloat16": ("<i2", torch.bfloat16), "int64": ("<i8", torch.int64)}


class _Memory:
    """A storage's device memory under the array interface that torch reads."""

    def __init__(self, storage):
        self.storage = storage  # the view keeps the memory alive
        self.__cuda_array_interface__ = {"shape": (storage.size,), "typestr": RAW[storage.dtype][0],
                                         "data": (storage.ptr, False), "strides": None, "version": 2}


def view(storage, shape):
    """The storage's memory as a torch tensor (no copy)."""
    return torch.as_tensor(_Memory(storage), device="cuda").view(RAW[storage.dtype][1]).reshape(shape)


def store(values):
    """A framework storage holding a torch tensor's values."""
    from qutai_amd.backends import amd

    storage = amd.AMDStorage(values.numel(), {raw[1]: name for name, raw in RAW.items()}[values.dtype])
    view(storage, values.shape).copy_(values)
    return storage


def tensor(values):
    from qutai_amd import Tensor

    return Tensor(store(values), shape=tuple(values.shape))


class Outputs(dict):
    """Named (storage, shape[, columns]) results, seen as torch tensors (no
    copy) when they are read: a program of this framework's users keeps the
    storages, so a pass does not pay for the conversion."""

    def __getitem__(self, name):
        storage, shape, *columns = super().__getitem__(name)
        values = view(storage, shape)
        return values[:, columns[0]:columns[1]] if columns else values


class Draws:
    """Random values on the GPU, from the seed alone."""

    def __init__(self, seed):
        self.generator = torch.Generator(device="cuda")
        self.generator.manual_seed(seed)

    def normal(self, shape, dtype="float32", std=1.0):
        return (torch.randn(shape, generator=self.generator, device="cuda") * std).to(TORCH[dtype])

    def uniform(self, shape, low=0.0, high=1.0):
        return torch.rand(shape, generator=self.generator, device="cuda") * (high - low) + low

    def integers(self, shape, low, high):
        return torch.randint(low, high, shape, generator=self.generator, device="cuda")


def log_between(rng, low, high):
    """An integer spread evenly over the logarithm; not only round ones."""
    return max(low, min(high, round(exp(rng.uniform(log(low), log(high))))))


# ---- norms of queries and keys per head, with the position rotation -------------------

class QueryKey:
    """RMSNorm of every head of q and k (a weight of the head's width each) and
    the rotation of its pairs (2i, 2i+1).  ``stacked``: q and k are columns of
    one projection product, beside v's, and so are their gradients.  ``past``:
    each sequence starts at a position of its own (a generation step)."""

    def inputs(self, c, seed):
        d, rows, dim = Draws(seed), c["batch"] * c["time"], c["dim"]
        wide_q, wide_k = c["heads"] * dim, c["kv_heads"] * dim
        x = {"wq": 1 + d.normal((dim,), std=0.1), "wk": 1 + d.normal((dim,), std=0.1)}
        if c["stacked"]:
            x["qkv"] = d.normal((rows, wide_q + 2 * wide_k), c["dtype"], 2.0)
            x["q"], x["k"] = x["qkv"][:, :wide_q], x["qkv"][:, wide_q:wide_q + wide_k]
        else:
            x["q"], x["k"] = d.normal((rows, wide_q), c["dtype"], 2.0), d.normal((rows, wide_k), c["dtype"], 0.5)
        if c["past"]:
            x["starts"] = d.integers((c["batch"],), c["past"] // 2, c["past"] + 1)
        if c["train"]:
            x["gq"], x["gk"] = d.normal((rows, wide_q), c["dtype"]), d.normal((rows, wide_k), c["dtype"])
        return x

    def prepare(self, c, x):
        if not own:
            return c, x
        return c, {n: store(v) for n, v in x.items() if not (c["stacked"] and n in "qk")}

    def run(self, state):
        c, x = state
        return self.framework(c, x) if own else self.plain(c, x)

    def framework(self, c, x):
        from qutai_amd.backends import amd, amd_lm

        rows, wide_q, wide_k = c["batch"] * c["time"], c["heads"] * c["dim"], c["kv_heads"] * c["dim"]
        dims = (c["batch"], c["time"], c["heads"], c["kv_heads"], c["dim"], THETA, EPS)
        row = wide_q + 2 * wide_k
        place = dict(q_row=row, k_column=wide_q, k_row=row) if c["stacked"] else {}
        place["starts"] = x.get("starts")
        q, k = (x["qkv"], x["qkv"]) if c["stacked"] else (x["q"], x["k"])
        out_q, out_k = amd_lm.qk_norm_rope(q, k, x["wq"], x["wk"], *dims, **place)
        out = Outputs(q=(out_q, (rows, wide_q)), k=(out_k, (rows, wide_k)))
        if not c["train"]:
            return out
        if c["stacked"]:  # into the columns of the gradient of the whole product
            block = amd.AMDStorage(rows * row, c["dtype"])
            _, _, dwq, dwk = amd_lm.qk_norm_rope_backward(x["gq"], x["gk"], q, k, x["wq"], x["wk"], *dims, **place,
                                                          out=block)
            out.update(dq=(block, (rows, row), 0, wide_q), dk=(block, (rows, row), wide_q, wide_q + wide_k))
        else:
            dq, dk, dwq, dwk = amd_lm.qk_norm_rope_backward(x["gq"], x["gk"], q, k, x["wq"], x["wk"], *dims, **place)
            out.update(dq=(dq, (rows, wide_q)), dk=(dk, (rows, wide_k)))
        out.update(dwq=(dwq, (c["dim"],)), dwk=(dwk, (c["dim"],)))
        return out

    def plain(self, c, x):
        at = torch.arange(c["time"], device="cuda", dtype=torch.float64)[None]
        at = at.expand(c["batch"], -1) if x.get("starts") is None else x["starts"][:, None] + at
        pairs = torch.arange(0, c["dim"], 2, device="cuda", dtype=torch.float64)
        angle = at.reshape(-1, 1, 1) * THETA ** (-pairs / c["dim"])
        cos, sin = angle.cos().float(), angle.sin().float()

        def rotated(values, sign):
            even, odd = values[..., 0::2], values[..., 1::2]
            return torch.stack((even * cos - sign * odd * sin, sign * even * sin + odd * cos), -1).flatten(-2)

        out = {}
        for name in ("q", "k"):
            weight = x["w" + name]
            rows = x[name].float().reshape(x[name].shape[0], -1, c["dim"])
            inverse = (rows.square().mean(-1, keepdim=True) + EPS).rsqrt()
            out[name] = rotated(rows * inverse * weight, 1).flatten(1).to(TORCH[c["dtype"]])
            if c["train"]:
                g = rotated(x["g" + name].float().reshape(rows.shape), -1)
                unit = rows * inverse
                t = g * weight
                dx = inverse * (t - unit * (t * unit).mean(-1, keepdim=True))
                out["d" + name] = dx.flatten(1).to(TORCH[c["dtype"]])
                out["dw" + name] = (g * unit).sum((0, 1))
        return out

    def exact(self, c, x):
        start = x["starts"].double() if c["past"] else torch.zeros(c["batch"], device="cuda", dtype=torch.float64)
        out = {}
        for name, heads in (("q", c["heads"]), ("k", c["kv_heads"])):
            rows = x[name].double().reshape(c["batch"], c["time"], heads, c["dim"]).clone().requires_grad_()
            weight = x["w" + name].double().requires_grad_()
            normed = weight * rows / (rows.pow(2).sum(-1, keepdim=True) / c["dim"] + EPS).sqrt()
            frequency = torch.exp(torch.arange(c["dim"] // 2, device="cuda", dtype=torch.float64)
                                  * (-2 * log(THETA) / c["dim"]))
            place = start[:, None] + torch.arange(c["time"], device="cuda", dtype=torch.float64)
            turn = torch.polar(torch.ones((), device="cuda", dtype=torch.float64),
                               place[:, :, None, None] * frequency)
            y = torch.view_as_real(torch.view_as_complex(normed.unflatten(-1, (-1, 2))) * turn)
            y = y.reshape(c["batch"] * c["time"], -1)
            out[name] = y.detach()
            if c["train"]:
                y.backward(x["g" + name].double())
                out["d" + name], out["dw" + name] = rows.grad.reshape(y.shape), weight.grad
        return out

    def work(self, c):
        values = c["batch"] * c["time"] * (c["heads"] + c["kv_heads"]) * c["dim"]
        return values * BYTES[c["dtype"]] * (5 if c["train"] else 2), values * (28 if c["train"] else 9)

    def draw(self, rng):
        heads = rng.choice([4, 8, 12, 16, 32])
        c = {"heads": heads, "kv_heads": heads // rng.choice([1, 2, 4]), "dim": rng.choice([32, 64, 64, 80, 96, 128, 128]),
             "dtype": rng.choice(["bfloat16", "bfloat16", "float32"]), "stacked": rng.random() < 0.6}
        if rng.random() < 0.4:
            return {**c, "batch": log_between(rng, 1, 256), "time": rng.choice([1, 1, 1, 2, 5]),
                    "past": log_between(rng, 10, 100000), "train": False}
        rows = 30_000_000 // ((heads + c["kv_heads"]) * c["dim"])
        batch = rng.randint(1, 8)
        return {**c, "batch": batch, "time": log_between(rng, 16, max(17, min(8192, rows // batch))), "past": 0,
                "train": rng.random() < 0.6}


# ---- a quantised key and value cache --------------------------------------------------

def groups_of(c):
    """Channels that share a scale: a row's, or 32 of them where codes have 4 bits."""
    return c["dim"] if c["bits"] == 8 else 32


def quantised(values, bits, group):
    """(codes, scales spread over the channels) of (..., dim) values: the scale
    is the smallest bfloat16 from 2^-100 up that keeps the group's codes within
    +-127 (+-7); codes are rounded to nearest, ties to even."""
    most = 127 if bits == 8 else 7
    dim = values.shape[-1]
    parts = -(-dim // group)
    wide = torch.nn.functional.pad(values.double(), (0, parts * group - dim)).unflatten(-1, (parts, group))
    scale = wide.abs().amax(-1, keepdim=True) / most
    # up to the next bfloat16: a double's fraction holds 45 bits more
    up = ((scale.view(torch.int64) + ((1 << 45) - 1)) >> 45 << 45).view(torch.float64).clamp(min=2.0 ** -100)
    scale = torch.where(scale.isfinite(), up, torch.nan)
    codes = torch.where(scale.isfinite(), (wide / scale).round(), 0.0)
    spread = scale.expand(wide.shape)
    return codes.flatten(-2)[..., :dim].to(torch.int8), spread.flatten(-2)[..., :dim].float()


def stands_for(values, bits, group):
    """The values that a quantised cache holds for ``values``, in 64 bits."""
    wide = values.double()
    out = torch.empty_like(wide)
    for start in range(0, wide.shape[-1], group):
        part = wide[..., start:start + group]
        scale = part.abs().amax(-1, keepdim=True) / (127 if bits == 8 else 7)
        fraction, exponent = torch.frexp(scale)  # 8 bits of significand, upwards
        power = ((exponent.long() + (1023 - 8)) << 52).view(torch.float64)  # 2^(exponent - 8), exactly
        scale = (torch.ceil(fraction * 256) * power).clamp(min=2.0 ** -100)
        out[..., start:start + group] = torch.round(part / scale) * scale
    return out


def channels(d, c):
    """The spread of the head channels' values: a few are much larger."""
    return torch.where(d.uniform((c["kv_heads"], c["dim"])) < 0.05, 8.0, 1.0) * d.uniform((c["kv_heads"], c["dim"]), 0.3, 1.5)


class CacheCopy:
    """A prompt's keys and values written into a quantised cache and read back."""

    def inputs(self, c, seed):
        d, shape = Draws(seed), (c["batch"], c["new"], c["kv_heads"], c["dim"])
        spread = channels(d, c)
        return {"k": (d.normal(shape) * spread).to(TORCH[c["dtype"]]), "v": d.normal(shape, c["dtype"])}

    def prepare(self, c, x):
        if not own:
            return c, x, None
        from qutai_amd.nn import QuantizedKVCache

        return c, {n: tensor(v) for n, v in x.items()}, QuantizedKVCache(c["new"], bits=c["bits"])

    def run(self, state):
        c, x, cache = state
        if own:
            cache.truncate(0)
            cache.append(x["k"], x["v"])
            keys, values = cache.read(c["dtype"])
            return Outputs(k=(keys.storage, keys.shape), v=(values.storage, values.shape))
        out = {}
        for name in "kv":
            codes, scales = quantised(x[name], c["bits"], groups_of(c))
            out[name] = (codes * scales).to(TORCH[c["dtype"]]).transpose(1, 2).contiguous()
        return out

    def exact(self, c, x):
        return {n: stands_for(x[n], c["bits"], groups_of(c)).transpose(1, 2).contiguous() for n in "kv"}

    def work(self, c):
        rows = 2 * c["batch"] * c["new"] * c["kv_heads"]
        held = c["dim"] * c["bits"] // 8 + 2 * -(-c["dim"] // groups_of(c))
        return rows * (2 * c["dim"] * BYTES[c["dtype"]] + 2 * held), rows * c["dim"] * 6

    def draw(self, rng):
        c = {"kv_heads": rng.choice([1, 2, 4, 8, 12, 16]), "dim": rng.choice([32, 40, 64, 64, 80, 96, 128, 128, 256]),
             "dtype": rng.choice(["bfloat16", "bfloat16", "float32"]), "bits": rng.choice([8, 8, 4])}
        rows = 16_000_000 // (c["kv_heads"] * c["dim"])
        batch = rng.randint(1, 16)
        return {**c, "batch": batch, "new": log_between(rng, 1, max(2, min(8000, rows // batch)))}


class CacheAttend:
    """New positions written into a quantised cache that holds ``past`` earlier
    ones at most (each sequence its own number), and their attention over it."""

    def inputs(self, c, seed):
        d, dim = Draws(seed), c["dim"]
        spread = channels(d, c)
        x = {}
        for name, length in (("old", c["past"]), ("new", c["new"])):
            shape = (c["batch"], length, c["kv_heads"], dim)
            x[name + "_k"] = (d.normal(shape) * spread).to(TORCH[c["dtype"]])
            x[name + "_v"] = d.normal(shape, c["dtype"])
        x["q"] = d.normal((c["batch"], c["new"], c["heads"], dim), c["dtype"], 1.5)
        if c["ragged"]:
            starts = d.integers((c["batch"],), c["past"] // 4, c["past"] + 1)
            starts[0] = c["past"]
            counts = d.integers((c["batch"],), c["new"] // 2, c["new"] + 1).clamp(min=1)
        else:
            starts = torch.full((c["batch"],), c["past"], device="cuda")
            counts = torch.full((c["batch"],), c["new"], device="cuda")
        return {**x, "starts": starts, "counts": counts}

    def prepare(self, c, x):
        starts, counts = x["starts"].tolist(), x["counts"].tolist()
        if own:
            from qutai_amd.nn import QuantizedKVCache

            cache = QuantizedKVCache(c["past"] + c["new"], bits=c["bits"])
            cache.append(tensor(x["old_k"]), tensor(x["old_v"]), starts)
            return c, starts, counts if min(counts) < c["new"] else None, cache, {n: tensor(x[n]) for n in ("new_k", "new_v", "q")}
        shape = (c["batch"], c["past"] + c["new"], c["kv_heads"], c["dim"])
        held = {}
        for name in "kv":
            codes, scales = (torch.zeros(shape, device="cuda", dtype=t) for t in (torch.int8, torch.float32))
            for b in range(c["batch"]):  # a sequence at a time: the 64-bit values are large
                codes[b, :c["past"]], scales[b, :c["past"]] = quantised(x["old_" + name][b], c["bits"], groups_of(c))
            held[name] = codes, scales
        return c, x["starts"], x["counts"], held, {n: x[n] for n in ("new_k", "new_v", "q")}

    def run(self, state):
        c, starts, counts, held, x = state
        if own:
            held.truncate(starts)
            held.append(x["new_k"], x["new_v"], counts)
            out = held.attend(x["q"])
            return Outputs(out=(out.storage, out.shape))
        new, kv_heads = c["new"], c["kv_heads"]
        steps = torch.arange(new, device="cuda")
        at, there = starts[:, None] + steps, steps < counts[:, None]
        sequence = torch.arange(c["batch"], device="cuda")[:, None].expand(at.shape)
        for name in "kv":
            for kept, fresh in zip(held[name], quantised(x["new_" + name], c["bits"], groups_of(c))):
                kept[sequence[there], at[there]] = fresh[there]
        k, v = ((codes * scales).transpose(1, 2) for codes, scales in (held["k"], held["v"]))
        q = x["q"].float().unflatten(2, (kv_heads, -1)).permute(0, 2, 4, 1, 3).flatten(3)  # channels x (new, group)
        scores = (k.contiguous() @ q.contiguous()).unflatten(3, (new, -1)) * c["dim"] ** -0.5
        hidden = torch.arange(k.shape[2], device="cuda")[:, None] > at[:, None, None, :]
        scores = scores.masked_fill(hidden[..., None], float("-inf"))
        weights = (scores - scores.amax(2, keepdim=True)).exp()
        sums = weights.sum(2)
        out = (weights.flatten(3).transpose(2, 3).contiguous() @ v.contiguous()).unflatten(2, (new, -1))
        out = (out / sums[..., None]).permute(0, 2, 1, 3, 4).flatten(2, 3)
        return {"out": torch.where(there[..., None, None], out, 0.0).to(TORCH[c["dtype"]])}

    def exact(self, c, x):
        group = c["heads"] // c["kv_heads"]
        out = torch.zeros(x["q"].shape, device="cuda", dtype=torch.float64)
        for b, (start, count) in enumerate(zip(x["starts"].tolist(), x["counts"].tolist())):
            for h in range(c["kv_heads"]):
                k, v = (stands_for(torch.cat((x["old_" + n][b, :start, h], x["new_" + n][b, :count, h])), c["bits"], groups_of(c))
                        for n in "kv")
                for g in range(h * group, (h + 1) * group):
                    scores = x["q"][b, :count, g].double() @ k.T.contiguous() / c["dim"] ** 0.5
                    later = torch.ones(scores.shape, device="cuda", dtype=torch.bool).triu(1 + start)
                    out[b, :count, g] = scores.masked_fill(later, float("-inf")).softmax(-1) @ v
        return {"out": out}

    def keys(self, c):
        """Visible keys of all sequences, and (query, key) pairs of a head."""
        fill = 0.625 if c["ragged"] else 1.0  # the mean of the drawn starts
        past, new = fill * c["past"], (0.75 if c["ragged"] else 1.0) * max(1, c["new"])
        return c["batch"] * (past + new), c["batch"] * new * (past + (new + 1) / 2)

    def work(self, c):
        held = c["dim"] * c["bits"] // 8 + 2 * -(-c["dim"] // groups_of(c))
        keys, pairs = self.keys(c)
        own_rows = c["batch"] * c["new"] * (2 * c["heads"] + 2 * c["kv_heads"]) * c["dim"] * BYTES[c["dtype"]]
        return int(2 * keys * c["kv_heads"] * held + own_rows), int(4 * pairs * c["heads"] * c["dim"])

    def draw(self, rng):
        kv_heads = rng.choice([1, 2, 4, 8, 8, 16])
        c = {"kv_heads": kv_heads, "heads": kv_heads * rng.choice([1, 1, 2, 4, 4, 8]),
             "dim": rng.choice([32, 40, 64, 64, 80, 96, 128, 128, 256]), "bits": rng.choice([8, 8, 4]),
             "dtype": rng.choice(["bfloat16", "bfloat16", "float32"]), "ragged": rng.random() < 0.6}
        if rng.random() < 0.3:  # a prompt, or a further part of one
            return {**c, "batch": rng.randint(1, 3), "heads": min(32, c["heads"]), "new": log_between(rng, 20, 500),
                    "past": rng.choice([0, 0, log_between(rng, 16, 3000)])}
        past = log_between(rng, 16, 20000)
        most = max(1, 200_000_000 // (past * kv_heads * c["dim"]))
        return {**c, "batch": log_between(rng, 1, min(64, most)) if most > 1 else 1, "new": rng.choice([1, 1, 1, 1, 2, 4, 7]), "past": past}


# ---- tokens from logits ---------------------------------------------------------------

class Sample:
    """One token for each row of logits: temperature, the top_k largest, the
    smallest set of these that holds top_p of their mass, those of at least
    min_p of the largest's weight, then the given number picks one.  ``mixed``:
    every row has parameters of its own (requests of many users)."""

    def inputs(self, c, seed):
        d, rows, vocab = Draws(seed), c["rows"], c["vocab"]
        logits = d.normal((rows, vocab), std=2.5)
        logits = torch.where(d.uniform((rows, vocab)) < 0.01, float("-inf"), logits).to(TORCH[c["dtype"]])  # banned tokens
        x = {"logits": logits, "uniforms": d.uniform((rows,))}
        if c["mixed"]:
            x["temperature"] = torch.where(d.uniform((rows,)) < 0.1, 0.0, d.uniform((rows,), 0.3, 1.3))
            x["top_k"] = torch.where(d.uniform((rows,)) < 0.5, 0, d.integers((rows,), 1, 200))
            x["top_p"] = torch.where(d.uniform((rows,)) < 0.3, 1.0, d.uniform((rows,), 0.5, 1.0))
            x["min_p"] = torch.where(d.uniform((rows,)) < 0.7, 0.0, d.uniform((rows,), 0.01, 0.1))
        return x

    PARAMETERS = ("temperature", "top_k", "top_p", "min_p")

    def prepare(self, c, x):
        state = {n: store(v) for n, v in x.items()} if own else dict(x)
        for name in self.PARAMETERS:
            if name in c:
                state[name] = c[name]
        return c, state

    def run(self, state):
        c, x = state
        if own:
            from qutai_amd.backends import amd_lm

            tokens, probabilities = amd_lm.sample(x["logits"], x["uniforms"], c["rows"], c["vocab"],
                                                  **{n: x[n] for n in self.PARAMETERS})
            return Outputs(tokens=(tokens, (c["rows"],)), probabilities=(probabilities, (c["rows"],)))
        column = [torch.as_tensor(x[n], device="cuda", dtype=torch.float64).expand(c["rows"])[:, None] for n in self.PARAMETERS]
        temperature, top_k, top_p, min_p = column
        logits = x["logits"].double()
        top = logits.amax(1, keepdim=True)
        weights = torch.where(temperature > 0, ((logits - top) / temperature.clamp(min=1e-30)).exp(), 0.0)
        ordered, order = torch.sort(x["logits"], dim=1, descending=True, stable=True)
        ordered = weights.gather(1, order)
        rank = torch.arange(c["vocab"], device="cuda")[None]
        ordered = torch.where((top_k > 0) & (rank >= top_k), 0.0, ordered)
        before = ordered.cumsum(1)
        enough = top_p * before[:, -1:]
        before = before - ordered
        kept = (ordered > 0) & ((rank == 0) | (top_p >= 1) | (before < enough)) & (ordered >= min_p)
        weights = torch.zeros_like(weights).scatter(1, order, torch.where(kept, ordered, 0.0))
        sums = weights.cumsum(1)
        token = (sums > x["uniforms"].double()[:, None] * sums[:, -1:]).to(torch.int8).argmax(1)
        token = torch.where(temperature[:, 0] > 0, token, order[:, 0])
        chance = weights.gather(1, token[:, None])[:, 0] / sums[:, -1]
        return {"tokens": token, "probabilities": torch.where(temperature[:, 0] > 0, chance, 1.0).float()}

    def exact(self, c, x):
        tokens, chances = [], []
        for r in range(c["rows"]):
            t, k, p, m = (float(x[n][r]) if n in x else float(c[n]) for n in self.PARAMETERS)
            row = x["logits"][r].double()
            order = torch.argsort(row, descending=True, stable=True)
            if t <= 0:
                tokens.append(order[0])
                chances.append(torch.ones((), device="cuda", dtype=torch.float64))
                continue
            kept = order[:int(k)] if k > 0 else order
            weight = torch.exp((row[kept] - row[order[0]]) / t)
            if p < 1:
                mass = torch.cumsum(weight, 0)
                kept = kept[:max(1, int(torch.searchsorted(mass, p * mass[-1])) + 1)]
            weight = torch.exp((row[kept] - row[order[0]]) / t)
            kept = torch.sort(kept[weight >= m]).values
            weight = torch.exp((row[kept] - row[order[0]]) / t)
            mass = torch.cumsum(weight, 0)
            at = torch.searchsorted(mass, x["uniforms"][r].double() * mass[-1], right=True).clamp(max=len(kept) - 1)
            tokens.append(kept[at])
            chances.append(weight[at] / mass[-1])
        return {"tokens": torch.stack(tokens), "probabilities": torch.stack(chances)}

    def work(self, c):
        return c["rows"] * (c["vocab"] * BYTES[c["dtype"]] + 16), c["rows"] * c["vocab"] * 6

    def draw(self, rng):
        vocab = rng.choice([1000, 8192, 32768, 32768, 49999, 65536, 131072, log_between(rng, 300, 131072)])
        c = {"vocab": vocab, "rows": log_between(rng, 1, min(256, 30_000_000 // vocab)),
             "dtype": rng.choice(["bfloat16", "float32"]), "mixed": rng.random() < 0.4}
        if c["mixed"]:
            return c
        return {**c, "temperature": rng.choice([0.0, 0.6, 0.8, 1.0, 1.0, 1.2]), "top_k": rng.choice([0, 0, 1, 20, 50, 400]),
                "top_p": rng.choice([1.0, 1.0, 0.9, 0.95, 0.5]), "min_p": rng.choice([0.0, 0.0, 0.05])}


KINDS = {"qk": QueryKey(), "copy": CacheCopy(), "attend": CacheAttend(), "sample": Sample()}


def listed():
    return [
        # a generation step's queries and keys, eight sequences at positions of their own: the smallest call
        {"name": "qk_step_bf16", "kind": "qk", "batch": 8, "time": 1, "heads": 16, "kv_heads": 4, "dim": 64,
         "dtype": "bfloat16", "stacked": True, "past": 1000, "train": False},
        # mixed-precision training of Config's attention: q and k as columns of one product, forward and backward
        {"name": "qk_train_bf16", "kind": "qk", "batch": 32, "time": 1024, "heads": 16, "kv_heads": 4, "dim": 64,
         "dtype": "bfloat16", "stacked": True, "past": 0, "train": True},
        # training in the default storage type, heads of an odd width, ragged rows
        {"name": "qk_train_fp32", "kind": "qk", "batch": 3, "time": 333, "heads": 12, "kv_heads": 12, "dim": 80,
         "dtype": "float32", "stacked": False, "past": 0, "train": True},
        # prompts written into the cache and read back
        {"name": "cache_copy_8bit", "kind": "copy", "batch": 4, "new": 4000, "kv_heads": 8, "dim": 128,
         "dtype": "bfloat16", "bits": 8},
        {"name": "cache_copy_4bit", "kind": "copy", "batch": 3, "new": 777, "kv_heads": 12, "dim": 80,
         "dtype": "float32", "bits": 4},
        # one sequence's generation step, where latency counts
        {"name": "attend_one", "kind": "attend", "batch": 1, "new": 1, "past": 1000, "heads": 16, "kv_heads": 4,
         "dim": 64, "dtype": "bfloat16", "bits": 8, "ragged": False},
        # a full batch of long sequences, each of its own length
        {"name": "attend_batch_8bit", "kind": "attend", "batch": 32, "new": 1, "past": 16000, "heads": 32, "kv_heads": 8,
         "dim": 128, "dtype": "bfloat16", "bits": 8, "ragged": True},
        {"name": "attend_batch_4bit", "kind": "attend", "batch": 16, "new": 1, "past": 8000, "heads": 32, "kv_heads": 8,
         "dim": 128, "dtype": "bfloat16", "bits": 4, "ragged": True},
        # a multi-head layer's step in the default storage type
        {"name": "attend_heads_fp32", "kind": "attend", "batch": 8, "new": 1, "past": 1001, "heads": 16, "kv_heads": 16,
         "dim": 64, "dtype": "float32", "bits": 8, "ragged": False},
        # a further part of two prompts over what the cache holds of them
        {"name": "attend_prompt", "kind": "attend", "batch": 2, "new": 512, "past": 3500, "heads": 16, "kv_heads": 4,
         "dim": 64, "dtype": "bfloat16", "bits": 8, "ragged": True},
        # one row of logits of Config's vocabulary
        {"name": "sample_one", "kind": "sample", "rows": 1, "vocab": 32768, "dtype": "float32", "mixed": False,
         "temperature": 0.8, "top_k": 50, "top_p": 0.95, "min_p": 0.0},
        # a serving batch, a large vocabulary, parameters of many users
        {"name": "sample_batch", "kind": "sample", "rows": 200, "vocab": 131072, "dtype": "bfloat16", "mixed": True},
    ]


def draw(rng):
    kind = rng.choice(sorted(KINDS))
    return {"kind": kind, **KINDS[kind].draw(rng)}


def prepare(case, seed):
    kind = KINDS[case["kind"]]
    return kind, kind.prepare(case, kind.inputs(case, seed))


def run(state):
    kind, inner = state
    return kind.run(inner)


def exact(case, seed):
    kind = KINDS[case["kind"]]
    return kind.exact(case, kind.inputs(case, seed))


def work(case):
    moved, flops = KINDS[case["kind"]].work(case)
    return {"bytes": moved, "flops": flops}
