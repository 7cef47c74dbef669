"""The operators of a training step over packed documents, as timed cases.

A case is a dict of plain values; its ``kind`` names one of the classes below:
attention of sequences of different lengths that lie one behind the other
(``attend``), rotary positions with a position for every token, in either
layout, over part of the head and with scaled frequencies (``rotate``), and an
AdamW step over many tensors with moments of 32 or 8 bits (``adamw``).  Sizes
are those of this repository's ``Config`` defaults (width 1024, 16 heads of 64
with 4 kv heads, SwiGLU 3584, vocabulary 32768, sequences of 1024) and generic
ones (32 heads of 128 with 8 kv heads, documents of thousands of tokens); odd
ones are mixed in by ``draw``.

``prepare`` draws the inputs on the GPU from the seed.  Where ``own`` is false
``run`` computes an operator from elementary torch operations in 32 bits (64
for angles, for the norm of all gradients and for moments that are held in 8
bits, where a value next to a border would change the result); where it is true
it calls the framework, which is then given the same values as its own
storages.  ``exact`` computes the outputs in 64 bits from the operators'
definitions.
"""
from __future__ import annotations

from math import exp, log, pi
from random import Random

import torch

own = False

TORCH = {"float32": torch.float32, "bfloat16": torch.bfloat16}
BYTES = {"float32": 4, "bfloat16": 2}


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


class Outputs(dict):
    """Named results that are made into torch tensors when they are read: a
    program keeps the framework's storages (and codes of 8 bits), so a pass does
    not pay for the conversion."""

    def __getitem__(self, name):
        return super().__getitem__(name)()


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


def lengths_of(c):
    """The case's documents: lengths spread over their logarithm up to the
    longest, which is among them, until they fill ``total`` tokens."""
    rng, left = Random(c["mix"]), c["total"]
    lengths = [min(c["longest"], left)]
    left -= lengths[0]
    while left > 0:
        lengths.append(min(left, log_between(rng, c["shortest"], c["longest"])))
        left -= lengths[-1]
    rng.shuffle(lengths)
    return lengths


# ---- attention over packed sequences --------------------------------------------------

class Attend:
    """Grouped-query attention of documents of different lengths, one behind the
    other in one matrix of tokens: every token sees its own document, up to
    itself where ``causal``.  ``stacked``: q, k and v are columns of one
    projection product.  ``train``: the gradients of q, k and v too."""

    def inputs(self, c, seed):
        d, rows, dim = Draws(seed), c["total"], c["dim"]
        wide_q, wide_k = c["heads"] * dim, c["kv_heads"] * dim
        if c["stacked"]:
            qkv = d.normal((rows, wide_q + 2 * wide_k), c["dtype"], 1.2)
            x = {"qkv": qkv, "q": qkv[:, :wide_q], "k": qkv[:, wide_q:wide_q + wide_k], "v": qkv[:, wide_q + wide_k:]}
        else:
            x = {"q": d.normal((rows, wide_q), c["dtype"], 1.5), "k": d.normal((rows, wide_k), c["dtype"]),
                 "v": d.normal((rows, wide_k), c["dtype"])}
        if c["train"]:
            x["g"] = d.normal((rows, wide_q), c["dtype"])
        return x

    def prepare(self, c, x):
        lengths = lengths_of(c)
        if own:
            from qutai_amd.lm import Packing

            return c, Packing(lengths), {n: store(v) for n, v in x.items() if not (c["stacked"] and n in ("q", "k", "v"))}
        starts = [0]
        for n in lengths:
            starts.append(starts[-1] + n)
        by_size = {}  # documents of similar lengths are padded to the longest of them
        for start, n in zip(starts, lengths):
            by_size.setdefault(max(0, n - 1).bit_length(), []).append((start, n))
        parts = []
        for group in by_size.values():
            start, n = (torch.tensor(column, device="cuda") for column in zip(*group))
            steps = torch.arange(max(n for _, n in group), device="cuda")
            there = steps < n[:, None]
            parts.append((torch.where(there, start[:, None] + steps, 0), there))
        return c, parts, x

    def run(self, state):
        c, plan, x = state
        return self.framework(c, plan, x) if own else self.plain(c, plan, x)

    def framework(self, c, packing, x):
        from qutai_amd.backends import amd_lm

        heads, kv_heads, dim, rows = c["heads"], c["kv_heads"], c["dim"], c["total"]
        wide_q, wide_k = heads * dim, kv_heads * dim
        row = wide_q + 2 * wide_k
        place = (dict(q_row=row, k_column=wide_q, k_row=row, v_column=wide_q + wide_k, v_row=row) if c["stacked"] else {})
        place["causal"] = c["causal"]
        q, k, v = (x["qkv"],) * 3 if c["stacked"] else (x["q"], x["k"], x["v"])
        if not c["train"]:
            out, _ = amd_lm.attention_packed(q, k, v, packing, heads, kv_heads, dim, **place)
            return Outputs(out=lambda: view(out, (rows, wide_q)))
        out, lse, rest = amd_lm.attention_packed(q, k, v, packing, heads, kv_heads, dim, **place, rest=True)
        dq, dk, dv = amd_lm.attention_packed_backward(x["g"], q, k, v, out, lse, packing, heads, kv_heads, dim, **place,
                                                      rest=rest)
        return Outputs(out=lambda: view(out, (rows, wide_q)), dq=lambda: view(dq, (rows, wide_q)),
                       dk=lambda: view(dk, (rows, wide_k)), dv=lambda: view(dv, (rows, wide_k)))

    def plain(self, c, parts, x):
        heads, kv_heads, dim = c["heads"], c["kv_heads"], c["dim"]
        names = ("out", "dq", "dk", "dv") if c["train"] else ("out",)
        result = {n: torch.empty((c["total"], (heads if n in ("out", "dq") else kv_heads) * dim), device="cuda",
                                 dtype=TORCH[c["dtype"]]) for n in names}
        for at, there in parts:
            documents, steps = at.shape

            def taken(name):  # (document, kv head, query heads of it x tokens, channels)
                rows = torch.where(there[..., None], x[name][at.flatten()].float().unflatten(0, at.shape), 0.0)
                rows = rows.unflatten(2, (kv_heads, -1, dim)).permute(0, 2, 3, 1, 4)
                return rows.reshape(documents, kv_heads, -1, dim).contiguous()

            def put(name, values):
                values = values.unflatten(2, (-1, steps)).permute(0, 3, 1, 2, 4).flatten(2)
                result[name][at[there]] = values[there].to(TORCH[c["dtype"]])

            q, k, v = taken("q"), taken("k"), taken("v")
            seen = there[:, None, None, None, :]
            if c["causal"]:
                seen = seen & torch.ones((steps, steps), device="cuda", dtype=torch.bool).tril()
            scores = (q @ k.transpose(2, 3).contiguous() * dim ** -0.5).unflatten(2, (-1, steps))
            scores = scores.masked_fill_(~seen, float("-inf"))
            weights = (scores - scores.amax(-1, keepdim=True)).exp_()
            del scores
            weights = (weights / weights.sum(-1, keepdim=True)).flatten(2, 3)
            out = weights @ v
            put("out", out)
            if c["train"]:
                g = taken("g")
                put("dv", weights.transpose(2, 3).contiguous() @ g)
                d = g @ v.transpose(2, 3).contiguous()
                d = weights.mul_(d.sub_((g * out).sum(-1, keepdim=True))).mul_(dim ** -0.5)
                put("dq", d @ k)
                put("dk", d.transpose(2, 3).contiguous() @ q)
        return result

    def exact(self, c, x):
        dim, group = c["dim"], c["heads"] // c["kv_heads"]
        names = {"out": "q", "dq": "q", "dk": "k", "dv": "v"} if c["train"] else {"out": "q"}
        out = {n: torch.zeros(x[like].shape, device="cuda", dtype=torch.float64) for n, like in names.items()}
        start = 0
        for n in lengths_of(c):
            rows = slice(start, start + n)
            later = torch.ones((n, n), device="cuda", dtype=torch.bool).triu(1)
            for h in range(c["kv_heads"]):
                of_kv, of_q = slice(h * dim, (h + 1) * dim), slice(h * group * dim, (h + 1) * group * dim)
                q = x["q"][rows, of_q].double().unflatten(1, (group, dim)).transpose(0, 1).contiguous()
                k, v = (x[m][rows, of_kv].double().contiguous() for m in "kv")
                scores = torch.matmul(q, k.T.contiguous()) / dim ** 0.5
                p = torch.softmax(scores.masked_fill(later, float("-inf")) if c["causal"] else scores, -1)
                del scores
                o = torch.matmul(p, v)
                out["out"][rows, of_q] = o.transpose(0, 1).flatten(1)
                if c["train"]:
                    g = x["g"][rows, of_q].double().unflatten(1, (group, dim)).transpose(0, 1).contiguous()
                    for j in range(group):
                        out["dv"][rows, of_kv] += p[j].T.contiguous() @ g[j]
                        ds = g[j] @ v.T.contiguous()
                        ds = p[j] * (ds - (ds * p[j]).sum(1, keepdim=True)) / dim ** 0.5
                        out["dk"][rows, of_kv] += ds.T.contiguous() @ q[j]
                        at = (h * group + j) * dim
                        out["dq"][rows, at:at + dim] = ds @ k
            start += n
        return out

    def work(self, c):
        pairs = sum(n * (n + 1) // 2 if c["causal"] else n * n for n in lengths_of(c))
        q, kv = c["total"] * c["heads"] * c["dim"], c["total"] * c["kv_heads"] * c["dim"]
        # forward q k v out; backward q k v out g and the three gradients
        values = (2 * q + 2 * kv) + ((4 * q + 4 * kv) if c["train"] else 0)
        return values * BYTES[c["dtype"]], pairs * c["heads"] * c["dim"] * (14 if c["train"] else 4)

    def draw(self, rng):
        kv_heads = rng.choice([1, 2, 4, 4, 8])
        c = {"kv_heads": kv_heads, "heads": kv_heads * rng.choice([1, 2, 3, 4, 4]),
             "dim": rng.choice([32, 40, 64, 64, 64, 80, 96, 128, 128, 128]),
             "dtype": rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"]), "causal": rng.random() < 0.8,
             "stacked": rng.random() < 0.5, "train": rng.random() < 0.65, "mix": rng.randrange(1 << 20)}
        longest = log_between(rng, 4, 4000 if c["dtype"] == "bfloat16" else 1500)
        most = min(16000, 40_000_000 // (c["heads"] * c["dim"]), 60_000_000_000 // (longest * c["heads"] * c["dim"]))
        return {**c, "longest": longest, "shortest": rng.choice([1, 1, max(1, longest // 8)]),
                "total": log_between(rng, longest, max(longest + 1, min(most, 400 * longest)))}


# ---- rotary positions -----------------------------------------------------------------

class Rotate:
    """The first ``rotary`` channels of every head of q and k turned by their
    token's position: pairs (2i, 2i+1) or, in the half layout, (i, i + rotary/2);
    pair i turns by theta^(-2i/rotary) radians a position, less where ``scaling``
    stretches the context by ``factor``.  ``past``: each sequence's tokens start
    at a position of its own (a generation step); else packed documents, which
    start theirs at 0 again.  ``stacked``: q and k are columns of one product,
    and their gradients of another."""

    THETA = 10000.0

    def inputs(self, c, seed):
        d, rows, dim = Draws(seed), c["total"], c["dim"]
        wide_q, wide_k = c["heads"] * dim, c["kv_heads"] * dim
        if c["stacked"]:
            qkv = d.normal((rows, wide_q + 2 * wide_k), c["dtype"], 2.0)
            x = {"qkv": qkv, "q": qkv[:, :wide_q], "k": qkv[:, wide_q:wide_q + wide_k]}
        else:
            x = {"q": d.normal((rows, wide_q), c["dtype"], 2.0), "k": d.normal((rows, wide_k), c["dtype"], 0.5)}
        if c["past"]:
            x["starts"] = d.integers((rows,), c["past"] // 2, c["past"] + 1)
        if c["train"]:
            x["gq"], x["gk"] = d.normal((rows, wide_q), c["dtype"]), d.normal((rows, wide_k), c["dtype"])
        return x

    def scaling(self, c):
        if c["scaling"] == "none":
            return None
        scaling = {"kind": c["scaling"], "factor": c["factor"]}
        return {**scaling, "original_length": 1024, "low": 1.0, "high": 32.0} if c["scaling"] == "parts" else scaling

    def prepare(self, c, x):
        if not own:
            if c["past"]:
                return c, x["starts"], x
            return c, torch.cat([torch.arange(n, device="cuda") for n in lengths_of(c)]), x
        from qutai_amd.lm import Packing, Rotary

        rotary = Rotary(c["dim"], self.THETA, rotary_dim=c["rotary"], layout=c["layout"], scaling=self.scaling(c))
        kept = {n: store(v) for n, v in x.items() if not (c["stacked"] and n in ("q", "k"))}
        return c, (rotary, None if c["past"] else Packing(lengths_of(c))), kept

    def run(self, state):
        c, plan, x = state
        return self.framework(c, plan, x) if own else self.plain(c, plan, x)

    def framework(self, c, plan, x):
        from qutai_amd.backends import amd, amd_lm

        rotary, packing = plan
        heads, kv_heads, dim, rows = c["heads"], c["kv_heads"], c["dim"], c["total"]
        wide_q, wide_k = heads * dim, kv_heads * dim
        row = wide_q + 2 * wide_k
        dims = (rotary, rows, 1, heads, kv_heads, dim) if c["past"] else (rotary, 1, rows, heads, kv_heads, dim)
        where = dict(starts=x["starts"]) if c["past"] else dict(positions=packing.positions)
        place = dict(q_row=row, k_column=wide_q, k_row=row) if c["stacked"] else {}
        q, k = (x["qkv"], x["qkv"]) if c["stacked"] else (x["q"], x["k"])
        out_q, out_k = amd_lm.rotary(q, k, *dims, **where, **place)
        out = Outputs(q=lambda: view(out_q, (rows, wide_q)), k=lambda: view(out_k, (rows, wide_k)))
        if c["train"] and c["stacked"]:  # into the columns of the gradient of the whole product
            block = amd.AMDStorage(rows * row, c["dtype"])
            amd_lm.rotary(x["gq"], x["gk"], *dims, **where, inverse=True, out=block, out_row=row, out_k_column=wide_q)
            out.update(dq=lambda: view(block, (rows, row))[:, :wide_q],
                       dk=lambda: view(block, (rows, row))[:, wide_q:wide_q + wide_k])
        elif c["train"]:
            dq, dk = amd_lm.rotary(x["gq"], x["gk"], *dims, **where, inverse=True)
            out.update(dq=lambda: view(dq, (rows, wide_q)), dk=lambda: view(dk, (rows, wide_k)))
        return out

    def plain(self, c, positions, x):
        r, dim = c["rotary"], c["dim"]
        at = torch.arange(0, r, 2, device="cuda", dtype=torch.float64) / r
        theta, magnitude = self.THETA, 1.0
        if c["scaling"] == "base":
            theta = theta * c["factor"] ** (r / (r - 2))
        frequency = theta ** -at
        if c["scaling"] == "linear":
            frequency = frequency / c["factor"]
        elif c["scaling"] == "parts":
            keep = ((1024 * frequency / (2 * pi) - 1.0) / 31.0).clamp(0, 1)
            frequency = frequency * (keep + (1 - keep) / c["factor"])
            magnitude = 0.1 * log(c["factor"]) + 1.0
        angle = positions.double()[:, None, None] * frequency
        cos, sin = (magnitude * angle.cos()).float(), (magnitude * angle.sin()).float()

        def turned(values, sign):
            values = values.float().reshape(c["total"], -1, dim)
            out, part = values.clone(), values[..., :r]
            if c["layout"] == "half":
                a, b = part[..., :r // 2], part[..., r // 2:]
                out[..., :r] = torch.cat((a * cos - sign * b * sin, sign * a * sin + b * cos), -1)
            else:
                a, b = part[..., 0::2], part[..., 1::2]
                out[..., :r] = torch.stack((a * cos - sign * b * sin, sign * a * sin + b * cos), -1).flatten(-2)
            return out.flatten(1).to(TORCH[c["dtype"]])

        out = {"q": turned(x["q"], 1), "k": turned(x["k"], 1)}
        if c["train"]:
            out.update(dq=turned(x["gq"], -1), dk=turned(x["gk"], -1))
        return out

    def exact(self, c, x):
        r, dim = c["rotary"], c["dim"]
        if c["past"]:
            places = x["starts"].double()
        else:
            places = torch.tensor([t for n in lengths_of(c) for t in range(n)], device="cuda", dtype=torch.float64)
        turns, magnitude = [], 1.0
        for i in range(r // 2):
            f = exp(-2 * i / r * log(self.THETA))
            if c["scaling"] == "base":
                f = exp(-2 * i / r * (log(self.THETA) + r / (r - 2) * log(c["factor"])))
            if c["scaling"] == "linear":
                f /= c["factor"]
            if c["scaling"] == "parts":
                kept = min(1.0, max(0.0, (1024 * f / (2 * pi) - 1.0) / (32.0 - 1.0)))
                f = kept * f + (1.0 - kept) * f / c["factor"]
                magnitude = 1.0 + 0.1 * log(c["factor"])
            turns.append(f)
        angle = places[:, None] * torch.tensor(turns, device="cuda", dtype=torch.float64)
        turn = torch.polar(torch.full_like(angle, magnitude), angle)[:, None]

        def rotated(values, factor):
            heads = values.double().reshape(c["total"], -1, dim).clone()
            pairs = (slice(0, r // 2), slice(r // 2, r)) if c["layout"] == "half" else (slice(0, r, 2), slice(1, r, 2))
            z = torch.complex(heads[..., pairs[0]].contiguous(), heads[..., pairs[1]].contiguous()) * factor
            heads[..., pairs[0]], heads[..., pairs[1]] = z.real, z.imag
            return heads.flatten(1)

        out = {"q": rotated(x["q"], turn), "k": rotated(x["k"], turn)}
        if c["train"]:
            out.update(dq=rotated(x["gq"], turn.conj()), dk=rotated(x["gk"], turn.conj()))
        return out

    def work(self, c):
        values = c["total"] * (c["heads"] + c["kv_heads"]) * c["dim"] * (2 if c["train"] else 1)
        return values * 2 * BYTES[c["dtype"]] + 8 * c["total"], values * 3 * c["rotary"] // c["dim"]

    def draw(self, rng):
        kv_heads = rng.choice([1, 2, 4, 8, 12])
        dim = rng.choice([32, 40, 64, 64, 80, 96, 128, 128, 256])
        c = {"kv_heads": kv_heads, "heads": kv_heads * rng.choice([1, 2, 4]), "dim": dim,
             "rotary": rng.choice([dim, dim, dim // 2, dim // 4 // 2 * 2]), "layout": rng.choice(["half", "half", "interleaved"]),
             "scaling": rng.choice(["none", "linear", "base", "parts"]), "factor": rng.choice([2.0, 4.0, 8.0, 7.5]),
             "dtype": rng.choice(["bfloat16", "bfloat16", "float32"]), "stacked": rng.random() < 0.6,
             "mix": rng.randrange(1 << 20)}
        if rng.random() < 0.35:
            return {**c, "total": log_between(rng, 1, 256), "past": log_between(rng, 10, 100000), "train": False}
        longest = log_between(rng, 16, 8192)
        most = max(longest + 1, min(65536, 100_000_000 // ((c["heads"] + kv_heads) * dim)))
        return {**c, "past": 0, "train": rng.random() < 0.7, "longest": longest, "shortest": rng.choice([1, max(1, longest // 8)]),
                "total": log_between(rng, longest, most)}


# ---- AdamW over many tensors --------------------------------------------------------------

MASK = (1 << 32) - 1
BLOCK = 256  # values that share an exponent


def mixed(x):
    """32 bits of each number, stirred (of a number or of an int64 tensor)."""
    x = x & MASK
    x = x ^ (x >> 15)
    x = (x * 0xBB67AE85) & MASK
    x = x ^ (x >> 13)
    x = (x * 0x6A09E667) & MASK
    return x ^ (x >> 16)


def dither(seed, step, tensor, count):
    """Two 16-bit numbers for each of a tensor's values at a step."""
    key = mixed(mixed(mixed(seed) + step) + tensor)
    bits = mixed(torch.arange(count, device="cuda", dtype=torch.int64) * 0x9E3779B9 + key)
    return bits & 0xFFFF, bits >> 16


def in_blocks(values):
    return torch.nn.functional.pad(values, (0, -values.numel() % BLOCK)).reshape(-1, BLOCK)


def power(exponent):
    """2^exponent in 64 bits, exactly (of an integer tensor)."""
    return ((exponent.long() + 1023) << 52).view(torch.float64)


def coded(values, bits, binades):
    """(codes, block exponents) of 64-bit values: magnitudes with three fraction
    bits in ``binades`` powers of two down from the block's exponent, rounded up
    where ``bits`` / 2^16 exceeds what is left of a step."""
    wide = in_blocks(values).abs()
    most = wide.amax(1, keepdim=True)
    fraction, exponent = torch.frexp(most)  # most = fraction 2^exponent, fraction in [1/2, 1)
    exponent = torch.where(most > 0, exponent - 1 + (fraction >= 0.9375), -64).clamp(min=-64)
    least = exponent - binades + 2  # the exponent of the lowest binade
    own_exponent = torch.where(wide > 0, torch.maximum(torch.frexp(wide)[1] - 1, least), least)
    steps = wide * power(3 - own_exponent) + in_blocks(bits) / 65536
    codes = (own_exponent - least) * 8 + steps.floor().long()
    return codes, exponent, least


def valued(codes, least):
    """The values that magnitude codes stand for, in 64 bits."""
    above = (codes >> 3).clamp(min=1) - 1
    return (codes - 8 * above).double() * power(least + above - 3)


class Moments8:
    """One tensor's moments in 8 bits: signs and magnitudes in 15 binades for the
    first, 31 binades for the second, in which a positive value keeps a code."""

    def __init__(self, count):
        self.count, blocks = count, -(-count // BLOCK)
        zeros = torch.zeros((blocks, BLOCK), device="cuda", dtype=torch.uint8)
        least = torch.zeros((blocks, 1), device="cuda", dtype=torch.int64)
        self.first, self.second = (zeros, zeros.bool(), least), (zeros, least)

    def read(self):
        codes, negative, least = self.first
        first = valued(codes.long(), least)
        second = valued(self.second[0].long(), self.second[1])
        return torch.where(negative, -first, first).flatten()[:self.count], second.flatten()[:self.count]

    def write(self, first, second, bits):
        codes, _, least = coded(first, bits[0], 16)
        self.first = codes.to(torch.uint8), in_blocks(first) < 0, least
        codes, _, least = coded(second, bits[1], 32)
        self.second = torch.where(in_blocks(second) > 0, codes.clamp(min=1), codes).to(torch.uint8), least


class AdamW:
    """A step over a model's tensors, the third of a run: m' = b1 m + (1 - b1) g,
    v' = b2 v + (1 - b2) g^2, p' = p (1 - lr decay) - lr m' / (1 - b1^t) /
    (sqrt(v' / (1 - b2^t)) + eps), with g scaled down where the norm of all
    gradients exceeds ``clip``.  ``bits``: what a moment is held in between
    steps."""

    LR, BETAS, EPS, DECAY, SEED, BEFORE = 3e-4, (0.9, 0.95), 1e-8, 0.1, 7, 2

    def shapes(self, c):
        if c["blocks"]:  # Config's blocks between its embedding and last norm, at a width of 1024 / shrink
            w = 1024 // c["shrink"]
            block = [w, w, w * w, w * w // 4, w * w // 4, w * w, w * w * 7 // 2, w * w * 7 // 2, w * w * 7 // 2]
            return [32768 // c["shrink"] * w] + block * c["blocks"] + [w]
        rng = Random(c["mix"])
        return [log_between(rng, 1, c["most"]) for _ in range(c["tensors"])]

    def inputs(self, c, seed):
        d, x = Draws(seed), {"p": [], "g": []}
        for i, n in enumerate(self.shapes(c)):
            x["p"].append(d.normal((n,), c["dtype"], 0.02))
            scale = 10.0 ** -(2.0 + 0.3 * (i % 7))
            gradients = []
            for _ in range(self.BEFORE + 1):
                g = d.normal((n,), std=scale)
                if i == 0:  # most of a vocabulary's rows are not in a batch
                    rows = d.uniform((-(-n // 64),)) < 0.7
                    g = torch.where(rows.repeat_interleave(64)[:n], 0.0, g)
                gradients.append(g.to(TORCH[c["dtype"]]))
            x["g"].append(gradients)
        return x

    def prepare(self, c, x):
        if own:
            from qutai_amd import Tensor
            from qutai_amd.optim import AdamW as Optimizer

            parameters = [Tensor(store(p), shape=tuple(p.shape), requires_grad=True) for p in x["p"]]
            optimizer = Optimizer(parameters, lr=self.LR, betas=self.BETAS, eps=self.EPS, weight_decay=self.DECAY,
                                  bits=c["bits"], max_norm=c["clip"] or None, seed=self.SEED)
            for k in range(self.BEFORE + 1):
                for p, g in zip(parameters, x["g"]):
                    p.grad = Tensor(store(g[k]), shape=tuple(p.shape))
                if k < self.BEFORE:
                    optimizer.step()
            return c, parameters, optimizer
        held = ([Moments8(p.numel()) for p in x["p"]] if c["bits"] == 8 else
                [tuple(torch.zeros(p.numel(), device="cuda") for _ in range(2)) for p in x["p"]])
        state = {"p": [p.clone() for p in x["p"]], "held": held, "step": 0}
        for k in range(self.BEFORE):
            state["g"] = [g[k] for g in x["g"]]
            self.plain(c, state)
        state["g"] = [g[self.BEFORE] for g in x["g"]]
        return c, state, None

    def run(self, state):
        c, inner, optimizer = state
        if not own:
            return self.plain(c, inner)
        optimizer.step()
        out = Outputs()
        for i, p in enumerate(inner):
            out[f"p{i}"] = lambda p=p: view(p.storage, p.shape)
            for name, moment in (("m", 0), ("v", 1)):
                out[f"{name}{i}"] = lambda p=p, moment=moment: view(optimizer.moments(p)[moment].storage, p.shape)
        return out

    def plain(self, c, state):
        b1, b2 = self.BETAS
        state["step"] += 1
        t, out, factor = state["step"], Outputs(), None
        if c["clip"]:
            norm = torch.stack([g.double().square().sum() for g in state["g"]]).sum().sqrt()
            factor = (c["clip"] / norm).clamp(max=1.0)
        for i, (p, g, held) in enumerate(zip(state["p"], state["g"], state["held"])):
            if c["bits"] == 8:
                g = g.double() if factor is None else g.double() * factor
                first, second = held.read()
                first, second = b1 * first + (1 - b1) * g, b2 * second + (1 - b2) * (g * g)
                held.write(first, second, dither(self.SEED, t, i, p.numel()))
                first, second = first.float(), second.float()
            else:
                g = g.float() if factor is None else g.float() * factor.float()
                first, second = held
                first.mul_(b1).add_((1 - b1) * g)
                second.mul_(b2).add_((1 - b2) * (g * g))
            update = (first / (1 - b1 ** t)) / ((second / (1 - b2 ** t)).sqrt() + self.EPS)
            p.copy_((p.float() - (self.LR * self.DECAY) * p.float() - self.LR * update).to(p.dtype))
            out[f"p{i}"] = lambda p=p: p
            for name, moment in (("m", 0), ("v", 1)):
                out[f"{name}{i}"] = (lambda held=held, moment=moment:
                                     held.read()[moment].float() if c["bits"] == 8 else held[moment])
        return out

    def exact(self, c, x):
        b1, b2 = self.BETAS
        p = [v.double() for v in x["p"]]
        held = [(torch.zeros_like(v), torch.zeros_like(v)) for v in p]
        for t in range(1, self.BEFORE + 2):
            gradients = [g[t - 1].double() for g in x["g"]]
            if c["clip"]:
                norm = sum(float(g.pow(2).sum()) for g in gradients) ** 0.5
                gradients = [g * min(1.0, c["clip"] / norm) for g in gradients]
            for i, g in enumerate(gradients):
                m, v = held[i][0] * b1 + g * (1 - b1), held[i][1] * b2 + g.pow(2) * (1 - b2)
                step = m / (1 - b1 ** t) / ((v / (1 - b2 ** t)).sqrt() + self.EPS)
                p[i] = (p[i] * (1 - self.LR * self.DECAY) - self.LR * step).to(TORCH[c["dtype"]]).double() \
                    if t <= self.BEFORE else p[i] * (1 - self.LR * self.DECAY) - self.LR * step
                if c["bits"] == 8:
                    low, high = dither(self.SEED, t, i, g.numel())
                    m, v = self.kept(m, low, 4, False), self.kept(v, high, 5, True)
                held[i] = m, v
        return {**{f"p{i}": v for i, v in enumerate(p)}, **{f"m{i}": h[0] for i, h in enumerate(held)},
                **{f"v{i}": h[1] for i, h in enumerate(held)}}

    def kept(self, values, bits, exponent_bits, positive):
        """What 8-bit codes hold of the values: the two neighbours of each on the
        grid of its block, and the upper one with the chance of its nearness."""
        powers = torch.tensor([2.0 ** k for k in range(-300, 300)], device="cuda", dtype=torch.float64)
        blocks = in_blocks(values)
        size = blocks.abs()
        top = size.amax(1, keepdim=True)
        binade = torch.searchsorted(powers, top, right=True) - 1  # the last power that is not above
        binade = (binade + (top >= 1.875 * powers[binade.clamp(min=0)]).long()).clamp(min=300 - 64)
        grid = powers[torch.maximum(torch.searchsorted(powers, size, right=True) - 1,
                                    binade - (2 ** exponent_bits - 2)) - 3]
        lower = torch.floor(size / grid) * grid
        up = (size - lower) / grid + in_blocks(bits).double() / 65536 >= 1
        held = lower + torch.where(up, grid, 0.0)
        if positive:
            held = torch.where((size > 0) & (held == 0), grid, held)
        return (held * torch.sign(blocks)).flatten()[:values.numel()]

    def work(self, c):
        count, item = sum(self.shapes(c)), BYTES[c["dtype"]]
        return count * (3 * item + (16 if c["bits"] == 32 else 4)), count * 14

    def draw(self, rng):
        c = {"bits": rng.choice([8, 8, 32]), "dtype": rng.choice(["float32", "float32", "bfloat16"]),
             "clip": rng.choice([0.0, 1.0, 0.25]), "blocks": 0, "mix": rng.randrange(1 << 20)}
        if rng.random() < 0.3:
            return {**c, "blocks": rng.randint(1, 2), "shrink": rng.choice([1, 2, 4, 8])}
        tensors = rng.randint(1, 20)
        return {**c, "tensors": tensors, "most": log_between(rng, 10, min(20_000_000, 60_000_000 // tensors))}


KINDS = {"attend": Attend(), "rotate": Rotate(), "adamw": AdamW()}


def listed():
    return [
        # a handful of short prompts read together: the smallest call
        {"name": "attend_few_bf16", "kind": "attend", "total": 90, "longest": 40, "shortest": 1, "mix": 3, "heads": 16,
         "kv_heads": 4, "dim": 64, "dtype": "bfloat16", "causal": True, "stacked": True, "train": False},
        # mixed-precision training of Config's attention on documents of up to its sequence length
        {"name": "attend_train_bf16", "kind": "attend", "total": 16384, "longest": 1024, "shortest": 16, "mix": 1,
         "heads": 16, "kv_heads": 4, "dim": 64, "dtype": "bfloat16", "causal": True, "stacked": True, "train": True},
        # training on long documents with wide heads
        {"name": "attend_long_bf16", "kind": "attend", "total": 16000, "longest": 6000, "shortest": 500, "mix": 2,
         "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bfloat16", "causal": True, "stacked": False, "train": True},
        # whole prompts of many users, answered next: forward alone
        {"name": "attend_prompts_bf16", "kind": "attend", "total": 6001, "longest": 2500, "shortest": 20, "mix": 5,
         "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bfloat16", "causal": True, "stacked": True, "train": False},
        # training in the default storage type, heads of an odd width, every token sees its whole document
        {"name": "attend_train_fp32", "kind": "attend", "total": 2999, "longest": 500, "shortest": 1, "mix": 4,
         "heads": 12, "kv_heads": 12, "dim": 80, "dtype": "float32", "causal": False, "stacked": False, "train": True},
        # a generation step of eight sequences at positions of their own
        {"name": "rotate_step_bf16", "kind": "rotate", "total": 8, "heads": 16, "kv_heads": 4, "dim": 64, "rotary": 64,
         "layout": "half", "scaling": "linear", "factor": 4.0, "dtype": "bfloat16", "stacked": True, "past": 4000,
         "train": False, "mix": 0},
        # packed training with wide heads and a context stretched by parts: columns of one product, forward and backward
        {"name": "rotate_train_bf16", "kind": "rotate", "total": 32768, "longest": 8192, "shortest": 64, "mix": 6,
         "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "layout": "half", "scaling": "parts", "factor": 8.0,
         "dtype": "bfloat16", "stacked": True, "past": 0, "train": True},
        # half of each head of an odd width, pairs side by side
        {"name": "rotate_train_fp32", "kind": "rotate", "total": 1001, "longest": 333, "shortest": 1, "mix": 7,
         "heads": 12, "kv_heads": 12, "dim": 80, "rotary": 40, "layout": "interleaved", "scaling": "base", "factor": 2.0,
         "dtype": "float32", "stacked": False, "past": 0, "train": True},
        # a small model's step, where latency counts
        {"name": "adamw_small_fp32", "kind": "adamw", "blocks": 2, "shrink": 16, "bits": 32, "dtype": "float32",
         "clip": 1.0, "mix": 0},
        # Config's embedding and two of its blocks
        {"name": "adamw_blocks_32bit", "kind": "adamw", "blocks": 2, "shrink": 1, "bits": 32, "dtype": "float32",
         "clip": 0.0, "mix": 0},
        {"name": "adamw_blocks_8bit", "kind": "adamw", "blocks": 2, "shrink": 1, "bits": 8, "dtype": "float32",
         "clip": 1.0, "mix": 0},
        # tensors of odd sizes held in bfloat16
        {"name": "adamw_odd_bf16", "kind": "adamw", "blocks": 0, "tensors": 17, "most": 3_000_001, "bits": 8,
         "dtype": "bfloat16", "clip": 0.0, "mix": 8},
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
