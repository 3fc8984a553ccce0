"""Operators of decoders in parts, as measurable cases.

A scene's surfels belong to parts (objects, packed scenes, experts), and a
part may have a decoder of its own, or a shared decoder with a low-rank
correction of its own. Each case is one pass through one operator:

* ``row_groups``: from each row's group, the order that puts the rows of a
  group together (stable; rows of no group last) and where each group begins;
* ``grouped``: a linear layer whose matrix and bias are those of the row's
  group, forward and backward or the forward alone; rows of no group give 0;
* ``adapted``: a linear layer that all rows share, plus ``scale`` times
  the product of two narrow matrices of the row's group, whose gradients and
  the rows' are taken (the shared matrix stays as it is), or the forward
  alone; rows of no group get the shared layer;
* ``dropout``: forward and backward, or the forward alone.

Row counts are the surfel counts of ``workloads.py`` (1,024 to a million)
and those of a few surfels decoded at a time; widths are generic. Parts are of
uneven sizes, some of them empty, and a hundredth of the rows are in none.

Dropout's mask: the Philox4x32-10 generator (Salmon, Moraes, Dror and Shaw,
"Parallel random numbers: as easy as 1, 2, 3", 2011) with the seed's two
words as its key and (column // 8, row's low word, row's high word, 0) as its
counter gives four words, 16 bits (low half first) to each of eight columns.
A value is kept where its bits are at least t = rint(65536 p), and multiplied
by 65536 / (65536 - t).
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}
SCALE = 0.5                            # of the low-rank correction
LIMIT_VALUES = 1_000_000 * 512         # rows * widest side of a drawn case
LIMIT_FLOPS = 6.0 * 1_000_000 * 512 * 512
LIMIT_WEIGHTS = 1 << 26                # values of all groups' matrices


def _case(name, op, rows, features=1, dtype="bfloat16", outputs=0, groups=0, rank=0, train=True,
          wide=False, p=0.0):
    return dict(name=name, op=op, rows=rows, features=features, dtype=dtype, outputs=outputs,
                groups=groups, rank=rank, train=train, wide=wide, p=p)


def listed():
    return [
        # A router's choice for each surfel of a mid-sized scene (64-bit
        # indices, as torch's argmax gives them).
        _case("groups_mid", "row_groups", 100_000, groups=64, wide=True),
        # The parts of the largest scene, many of them.
        _case("groups_large", "row_groups", 1_000_000, groups=512),
        # A few surfels decoded (picking, editing), each by its part's matrix.
        _case("grouped_rows", "grouped", 4, 1_024, outputs=1_024, groups=8, train=False),
        # The heads that give the neural renderer's 57 values, one to a part,
        # in its type: launches and host time count.
        _case("grouped_small", "grouped", 1_024, 64, "float32", outputs=57, groups=16),
        # A hidden layer of a mid-sized scene's parts.
        _case("grouped_mid", "grouped", 100_000, 256, outputs=256, groups=64),
        # Many small parts: as many weights as rows' values.
        _case("grouped_many", "grouped", 50_000, 128, "float16", outputs=128, groups=512),
        # A hidden layer of the largest scene.
        _case("grouped_large", "grouped", 1_000_000, 512, outputs=512, groups=32),
        # A few surfels of many scenes decoded at once.
        _case("adapted_rows", "adapted", 8, 1_024, outputs=1_024, groups=16, rank=16,
              train=False),
        # A head whose widths no vector load divides.
        _case("adapted_odd", "adapted", 33_333, 187, "float16", outputs=57, groups=7, rank=5),
        # A hidden layer of the largest scene fitted to its parts.
        _case("adapted_large", "adapted", 1_000_000, 512, outputs=512, groups=64, rank=16),
        # Hidden values of a small scene, in the renderer's own type.
        _case("dropout_small", "dropout", 10_000, 128, "float32", p=0.1),
        # Hidden values of the largest scene.
        _case("dropout_large", "dropout", 1_000_000, 512, p=0.2),
    ]


def _log(rng, low, high):
    return int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))


def draw(rng):
    """Any operator, type and size between the listed ones, odd ones among
    them."""
    while True:
        op = rng.choice(("row_groups", "grouped", "grouped", "adapted", "adapted", "dropout"))
        rows = _log(rng, 1, 1_000_000)
        dtype = rng.choice(("float32", "bfloat16", "bfloat16", "float16"))
        case = _case("", op, rows, dtype=dtype)
        del case["name"]
        if op == "row_groups":
            case.update(groups=_log(rng, 1, 512), wide=rng.random() < 0.5)
            return case
        case.update(features=rng.choice((_log(rng, 8, 1_024), 32 * _log(rng, 1, 32))),
                    train=rng.random() < 0.8)
        if op == "dropout":
            case["p"] = rng.choice((0.1, 0.25, rng.random()))
        else:
            case.update(outputs=rng.choice((18, 57, _log(rng, 8, 1_024),
                                            32 * _log(rng, 1, 32))),
                        groups=_log(rng, 1, 512))
        if op == "adapted":
            case["rank"] = rng.choice((4, 8, 16, 32, _log(rng, 1, 64)))
        elif op == "grouped" and \
                case["groups"] * case["outputs"] * case["features"] > LIMIT_WEIGHTS:
            continue
        if rows * max(case["features"], case["outputs"]) <= LIMIT_VALUES and \
                work(case)["flops"] <= LIMIT_FLOPS:
            return case


def work(case):
    rows, features, outputs = case["rows"], case["features"], case["outputs"]
    groups, rank, size = case["groups"], case["rank"], BYTES[case["dtype"]]
    plan = 4 * rows + 4 * (groups + 1)  # the order of the rows, the groups' beginnings
    if case["op"] == "row_groups":
        return {"bytes": rows * (8 if case["wide"] else 4) + plan, "flops": rows}
    passes = 2 if case["train"] else 1
    if case["op"] == "dropout":
        return {"bytes": passes * 2 * rows * features * size,
                "flops": passes * 16 * rows * features}
    sides = passes * rows * (features + outputs) * size
    if case["op"] == "grouped":
        parameters = passes * groups * outputs * (features + 1) * size
        return {"bytes": sides + parameters + plan,
                "flops": (6 if case["train"] else 2) * rows * features * outputs}
    parameters = (outputs * (features + 1) + passes * groups * rank * (features + outputs)) * size
    narrow = (6 if case["train"] else 2) * rows * rank * (features + outputs)
    return {"bytes": sides + parameters + plan,
            "flops": passes * 2 * rows * features * outputs + narrow}


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)
    rows, features, groups = case["rows"], case["features"], case["groups"]
    dtype = DTYPES[case["dtype"]]
    state = dict(case=case)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=device)

    def uniform(*shape):
        return torch.rand(shape, generator=gen, device=device) * 2 - 1

    if groups:
        # Parts whose sizes differ by several times, a tenth of them empty
        # where there are ten; a hundredth of the rows in none.
        shares = torch.exp(normal(groups))
        shares[1::10] *= 0 if groups >= 10 else 1
        index = torch.multinomial(shares, rows, replacement=True, generator=gen)
        index[uniform(rows) > 0.98] = -1
        state["index"] = index if case["wide"] else index.to(torch.int32)
        if case["op"] != "row_groups":
            # Parts stay as they are while they are decoded and fitted: a
            # program sorts the surfels by part once.
            key = torch.where(index < 0, groups, index)
            state["order"] = torch.argsort(key, stable=True).to(torch.int32)
            counts = torch.bincount(key, minlength=groups + 1)
            state["offsets"] = (torch.cumsum(counts, 0) - counts).to(torch.int32)
        else:
            return state
    x = normal(rows, features)
    grads = (rows, features)
    if case["op"] == "dropout":
        state["seed"] = (seed * 0x9E3779B1 + 12345) % (1 << 63)
    else:
        outputs, rank = case["outputs"], case["rank"]
        shape = (groups, outputs) if case["op"] == "grouped" else (outputs,)
        state["weight"] = (uniform(*shape, features) / math.sqrt(features)).to(dtype)
        state["bias"] = (uniform(*shape) / math.sqrt(features)).to(dtype)
        if rank:
            state["down"] = (uniform(groups, rank, features) / math.sqrt(features)).to(dtype)
            state["up"] = (uniform(groups, outputs, rank) / math.sqrt(rank)).to(dtype)
        grads = (rows, outputs)
    state["x"] = x.to(dtype)
    del x
    if case["train"]:
        state["grad"] = (normal(*grads) * 0.05).to(dtype)
        for name in _trained(case):
            state[name].requires_grad_()
    return state


def _trained(case):
    return {"dropout": ("x",), "grouped": ("x", "weight", "bias"),
            "adapted": ("x", "down", "up")}[case["op"]]


# --------------------------------------------------------------------------
# The operators in their plain form


def _plain_groups(state):
    groups = state["case"]["groups"]
    index = state["index"].long()
    key = torch.where((index < 0) | (index >= groups), groups, index)
    order = torch.argsort(key, stable=True).to(torch.int32)
    offsets = torch.searchsorted(key[order], torch.arange(groups + 1, device=key.device))
    return {"order": order, "offsets": offsets.to(torch.int32)}


class _Blocks:
    """The rows as blocks of ``size`` rows of one group, so that one batched
    product takes all groups: ``group`` [blocks] and ``rows`` [blocks, size],
    both one past the last where there is nothing."""

    def __init__(self, state):
        case, offsets, order = state["case"], state["offsets"].long(), state["order"].long()
        groups, rows = case["groups"], case["rows"]
        self.size = min(1024, max(16, rows // groups // 2))
        begin, end = offsets[:-1], offsets[1:]
        last = torch.cumsum((end - begin + self.size - 1) // self.size, 0)
        first = last - (end - begin + self.size - 1) // self.size
        block = torch.arange(rows // self.size + groups, device=order.device)
        self.group = torch.searchsorted(last, block, right=True)
        of = self.group.clamp_max(groups - 1)
        at = (begin[of] + (block - first[of]) * self.size)[:, None] + \
            torch.arange(self.size, device=order.device)
        inside = (self.group < groups)[:, None] & (at < end[of][:, None])
        self.rows = torch.where(inside, order[at.clamp(0, rows - 1)], rows)
        self.count, self.groups = rows, groups

    def take(self, values):
        """[blocks, size, width] float32, zero where there is no row."""
        values = values.float()
        return torch.cat((values, values.new_zeros(1, values.shape[1])))[self.rows]

    def put(self, blocks):
        """Rows from blocks; zero for a row of no group."""
        out = blocks.new_zeros(self.count + 1, blocks.shape[2])
        out[self.rows.reshape(-1)] = blocks.reshape(-1, blocks.shape[2])
        return out[:self.count]

    def of(self, matrices):
        """Each block's matrix, float32."""
        return matrices.float()[self.group.clamp_max(self.groups - 1)]

    def sum(self, blocks):
        """[groups, ...]: the sum over each group's blocks."""
        out = blocks.new_zeros(self.groups + 1, *blocks.shape[1:])
        return out.index_add_(0, self.group, blocks)[:self.groups]


def _turned(matrices):
    return matrices.transpose(1, 2).contiguous()


def _plain_grouped(state):
    x, weight, bias = state["x"], state["weight"], state["bias"]
    blocks = _Blocks(state)
    taken, matrices = blocks.take(x), blocks.of(weight)
    y = torch.bmm(taken, _turned(matrices)) + blocks.of(bias)[:, None]
    y = blocks.put(y).to(x.dtype)
    if not state["case"]["train"]:
        return {"y": y}
    g = blocks.take(state["grad"])
    return {"y": y, "dx": blocks.put(torch.bmm(g, matrices)).to(x.dtype),
            "dweight": blocks.sum(torch.bmm(_turned(g), taken)).to(x.dtype),
            "dbias": blocks.sum(g.sum(1)).to(x.dtype)}


def _plain_adapted(state):
    x, w32 = state["x"], state["weight"].float()
    blocks = _Blocks(state)
    taken, down, up = blocks.take(x), blocks.of(state["down"]), blocks.of(state["up"])
    inner = torch.bmm(taken, _turned(down))
    y = x.float() @ w32.t() + state["bias"].float()
    y = (y + SCALE * blocks.put(torch.bmm(inner, _turned(up)))).to(x.dtype)
    if not state["case"]["train"]:
        return {"y": y}
    g = blocks.take(state["grad"])
    back = torch.bmm(g, up)
    dx = state["grad"].float() @ w32 + SCALE * blocks.put(torch.bmm(back, down))
    return {"y": y, "dx": dx.to(x.dtype),
            "ddown": (SCALE * blocks.sum(torch.bmm(_turned(back), taken))).to(x.dtype),
            "dup": (SCALE * blocks.sum(torch.bmm(_turned(g), inner))).to(x.dtype)}


_WORD = 0xFFFFFFFF


def _philox(c0, c1, c2, c3, k0, k1):
    """Ten rounds on int64 tensors that hold 32-bit words; k0 and k1 are
    numbers."""
    for _ in range(10):
        # The products wrap modulo 2^64, and their words are masked out.
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (((b >> 32) & _WORD) ^ c1 ^ k0, b & _WORD,
                          ((a >> 32) & _WORD) ^ c3 ^ k1, a & _WORD)
        k0, k1 = (k0 + 0x9E3779B9) & _WORD, (k1 + 0xBB67AE85) & _WORD
    return c0, c1, c2, c3


def _plain_dropout(state):
    case, x, seed = state["case"], state["x"], state["seed"]
    rows, features = case["rows"], case["features"]
    chunk = torch.arange((features + 7) // 8, device=x.device)[None, :].expand(rows, -1)
    row = torch.arange(rows, device=x.device)[:, None].expand_as(chunk)
    words = _philox(chunk, row & _WORD, row >> 32, torch.zeros_like(row), seed & _WORD,
                    (seed >> 32) & _WORD)
    bits = torch.stack([half for word in words for half in (word & 0xFFFF, word >> 16)], -1)
    least = round(65536 * case["p"])
    keep = bits.reshape(rows, -1)[:, :features] >= least
    scale = 65536 / (65536 - least) if least < 65536 else 0.0
    y = torch.where(keep, x.float() * scale, 0.0).to(x.dtype)
    if not case["train"]:
        return {"y": y}
    return {"y": y, "dx": torch.where(keep, state["grad"].float() * scale, 0.0).to(x.dtype)}


# --------------------------------------------------------------------------
# The framework's operators


def _own_call(state):
    from diff_gabor_splatting_amd import layers

    case = state["case"]
    if case["op"] == "dropout":
        return layers.dropout(state["x"], case["p"], state["seed"])
    groups = layers.RowGroups(state["offsets"], state["order"])
    if case["op"] == "grouped":
        return layers.grouped_linear(state["x"], state["weight"], groups, state["bias"])
    return layers.adapted_linear(state["x"], state["weight"], state["down"], state["up"], groups,
                                 state["bias"], scale=SCALE)


def _own_groups(state):
    from diff_gabor_splatting_amd import layers

    groups = layers.row_groups(state["index"], state["case"]["groups"])
    return {"order": groups.order, "offsets": groups.offsets}


def run(state):
    case = state["case"]
    if not own:
        with torch.no_grad():
            return {"row_groups": _plain_groups, "grouped": _plain_grouped,
                    "adapted": _plain_adapted, "dropout": _plain_dropout}[case["op"]](state)
    if case["op"] == "row_groups":
        return _own_groups(state)
    if not case["train"]:
        with torch.no_grad():
            return {"y": _own_call(state)}
    y = _own_call(state)
    names = _trained(case)
    grads = torch.autograd.grad(y, [state[name] for name in names], state["grad"])
    return {"y": y, **{"d" + name: grad for name, grad in zip(names, grads)}}


# --------------------------------------------------------------------------
# The operators' definition in 64 bits


def _kept(seed, rows, features, least, device):
    """Which values the generator keeps, word by word in 64-bit halves of a
    32 x 32 product."""
    def product(a, m):  # high and low word of a * m, in 16-bit limbs
        low, high = (a & 0xFFFF) * m, (a >> 16) * m
        middle = high + (low >> 16)
        return middle >> 16, ((middle & 0xFFFF) << 16) | (low & 0xFFFF)

    out = torch.empty(rows, features, dtype=torch.bool, device=device)
    for first in range(0, rows, 1 << 16):
        row = torch.arange(first, min(rows, first + (1 << 16)), device=device)[:, None]
        column = torch.arange(0, features, 8, device=device)[None, :]
        counter = [column + 0 * row, row % (1 << 32) + 0 * column, row // (1 << 32) + 0 * column,
                   0 * row + 0 * column]
        counter[0] = counter[0] // 8
        key = [seed % (1 << 32), seed // (1 << 32) % (1 << 32)]
        for number in range(10):
            high0, low0 = product(counter[0], 0xD2511F53)
            high1, low1 = product(counter[2], 0xCD9E8D57)
            k0 = (key[0] + number * 0x9E3779B9) % (1 << 32)
            k1 = (key[1] + number * 0xBB67AE85) % (1 << 32)
            counter = [high1 ^ counter[1] ^ k0, low1, high0 ^ counter[3] ^ k1, low0]
        for j in range(8):
            part = out[first:first + (1 << 16), j::8]
            bits = (counter[j // 2] // (65536 if j % 2 else 1)) % 65536
            part.copy_((bits >= least)[:, :part.shape[1]])
    return out


def exact(case, seed):
    state = {k: v.detach() if isinstance(v, torch.Tensor) else v
             for k, v in prepare(case, seed).items()}
    if case["op"] == "row_groups":
        return None
    x = state["x"].double()
    g = state["grad"].double() if case["train"] else None
    if case["op"] == "dropout":
        least = round(65536 * case["p"])
        keep = _kept(state["seed"], case["rows"], case["features"], least, x.device)
        scale = 65536 / max(65536 - least, 1)
        out = {"y": x.mul_(scale).masked_fill_(~keep, 0)}
        if case["train"]:
            out["dx"] = g.mul_(scale).masked_fill_(~keep, 0)
        return out
    members = [torch.nonzero(state["index"] == group).flatten()
               for group in range(case["groups"])]
    weight, bias = state["weight"].double(), state["bias"].double()
    if case["op"] == "grouped":
        out = {"y": x.new_zeros(case["rows"], case["outputs"])}
        if case["train"]:
            out.update(dx=torch.zeros_like(x), dweight=torch.zeros_like(weight),
                       dbias=torch.zeros_like(bias))
        for group, rows in enumerate(members):
            if len(rows) == 0:
                continue
            part = x[rows]
            out["y"][rows] = torch.addmm(bias[group], part, weight[group].t())
            if case["train"]:
                out["dx"][rows] = torch.mm(g[rows], weight[group])
                out["dweight"][group] = torch.mm(g[rows].t(), part)
                out["dbias"][group] = g[rows].sum(0)
        return out
    down, up = state["down"].double(), state["up"].double()
    out = {"y": torch.addmm(bias, x, weight.t())}
    if case["train"]:
        out.update(dx=torch.mm(g, weight), ddown=torch.zeros_like(down),
                   dup=torch.zeros_like(up))
    for group, rows in enumerate(members):
        if len(rows) == 0:
            continue
        low_rank = torch.mm(up[group], down[group]) * SCALE  # [outputs, features]
        part = x[rows]
        out["y"][rows] += torch.mm(part, low_rank.t())
        if case["train"]:
            out["dx"][rows] += torch.mm(g[rows], low_rank)
            # The gradient of the product of both, [outputs, features].
            whole = torch.mm(g[rows].t(), part) * SCALE
            out["ddown"][group] = torch.mm(up[group].t(), whole)
            out["dup"][group] = torch.mm(whole, down[group].t())
    return out
